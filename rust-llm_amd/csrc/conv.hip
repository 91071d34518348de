// C ABI of the short causal convolution (include/rl_mixers.h); the kernel is in conv.h.
#include <hip/hip_runtime.h>

#include <new>
#include <string>
#include <vector>

#include "conv.h"
#include "mix_args.h"

using namespace rl;

struct rl_conv {
    int device = 0;
    uint32_t channels = 0, width = 0, activation = 0;
    float *weight = nullptr; // [width][channels], then the biases
    ~rl_conv() { (void)hipFree(weight); }
};

namespace {

// Rows of a run: the least that holds the longest state. The rows that are read again are still in the L2 and short runs
// give many waves; us with runs of 8 / 16 / 32, bf16, width 4: 512 x 8192 6.0 / 7.8 / 11.4, 2048 x 8192 14.8 / 14.9 / 17.8,
// 8192 x 8192 44.3 / 47.7 / 47.2, 8192 x 5120 32.1 / 31.8 / 30.7; width 8 51.1 / 56.6 / 57.1; f32, 1024 x 2027 7.1 / 10.0 / 15.0.
constexpr uint32_t CONV_RUN = CONV_MAX_WIDTH;

template <typename T, int W, bool WIDE>
void launch_conv(const ConvArgs &a, uint32_t blocks, bool silu, hipStream_t s) {
    if (silu) hipLaunchKernelGGL((k_conv<T, W, WIDE, true>), dim3(blocks), dim3(CONV_LANES), 0, s, a);
    else hipLaunchKernelGGL((k_conv<T, W, WIDE, false>), dim3(blocks), dim3(CONV_LANES), 0, s, a);
}

template <typename F>
void with_width(uint32_t width, F f) {
    switch (width) {
    case 2: return f(std::integral_constant<int, 2>{});
    case 3: return f(std::integral_constant<int, 3>{});
    case 4: return f(std::integral_constant<int, 4>{});
    case 5: return f(std::integral_constant<int, 5>{});
    case 6: return f(std::integral_constant<int, 6>{});
    case 7: return f(std::integral_constant<int, 7>{});
    default: return f(std::integral_constant<int, 8>{});
    }
}

}  // namespace

extern "C" {

int rl_conv_create(int device, uint32_t channels, uint32_t width, const float *weight, const float *bias,
                   uint32_t activation, rl_conv **out) {
    if (!out) return fail(RL_ERR_ARGUMENT, "out is null");
    *out = nullptr;
    if (!weight) return fail(RL_ERR_ARGUMENT, "weight is null");
    if (channels == 0) return fail(RL_ERR_ARGUMENT, "channels must be positive");
    if (width < 2 || width > CONV_MAX_WIDTH) return fail(RL_ERR_ARGUMENT, "width must be from 2 to 8");
    if (activation > RL_CONV_SILU) return fail(RL_ERR_ARGUMENT, "unknown activation");
    if (channels > 1u << 20) return fail(RL_ERR_CAPACITY, "more than 2^20 channels");
    DeviceGuard guard(device);
    if (!guard.ok) return fail(RL_ERR_DEVICE, "cannot select device " + std::to_string(device));
    auto *h = new (std::nothrow) rl_conv();
    if (!h) return fail(RL_ERR_CAPACITY, "out of host memory");
    h->device = device;
    h->channels = channels, h->width = width, h->activation = activation;
    const size_t size = (size_t)(width + 1) * channels;
    float *laid = new (std::nothrow) float[size];
    if (!laid) {
        delete h;
        return fail(RL_ERR_CAPACITY, "out of host memory");
    }
    for (uint32_t c = 0; c < channels; c++) {
        for (uint32_t j = 0; j < width; j++) laid[(size_t)j * channels + c] = weight[(size_t)c * width + j];
        laid[(size_t)width * channels + c] = bias ? bias[c] : 0.0f;
    }
    hipError_t e = hipMalloc(&h->weight, size * sizeof(float));
    if (e == hipSuccess) e = hipMemcpy(h->weight, laid, size * sizeof(float), hipMemcpyHostToDevice);
    delete[] laid;
    if (e != hipSuccess) {
        delete h;
        return hip_fail(e, "rl_conv_create");
    }
    *out = h;
    return RL_OK;
}

void rl_conv_destroy(rl_conv *conv) {
    if (!conv) return;
    DeviceGuard guard(conv->device);
    delete conv;
}

int rl_conv_rows(rl_conv *h, const rl_heads *x, const rl_heads *out, void *states, uint64_t state_slots,
                 const int32_t *slots_in, const int32_t *slots_out, const int32_t *starts, uint32_t rows, uint32_t seqs,
                 void *stream) {
    if (!h) return fail(RL_ERR_ARGUMENT, "conv is null");
    CHECK_HEADS(x, "x", false);
    CHECK_HEADS(out, "out", true);
    if (x->heads != 1 || out->heads != 1 || x->dim != h->channels || out->dim != h->channels)
        return fail(RL_ERR_ARGUMENT, "x and out must be one head of the handle's channels");
    if (x->dtype != out->dtype) return fail(RL_ERR_ARGUMENT, "x and out differ in type");
    if (rows && x->data == out->data) return fail(RL_ERR_ARGUMENT, "out must not be x");
    if (!starts && seqs != rows) return fail(RL_ERR_ARGUMENT, "without starts there is one row a sequence");
    if (rows && !seqs) return fail(RL_ERR_ARGUMENT, "rows without a sequence");
    if (seqs == 0) return RL_OK;
    if (!slots_in || !slots_out) return fail(RL_ERR_ARGUMENT, "slots_in and slots_out must be device pointers");
    if (state_slots && !states) return fail(RL_ERR_ARGUMENT, "states must be a device pointer");
    if ((uintptr_t)states % type_bytes(x->dtype)) return fail(RL_ERR_ARGUMENT, "states is not aligned to its type");
    if (rows > MAX_ROWS || seqs > MAX_ROWS) return fail(RL_ERR_CAPACITY, "more than 2^23 rows or sequences in a call");
    DeviceGuard guard(h->device);
    if (!guard.ok) return fail(RL_ERR_DEVICE, "cannot select the handle's device");
    ConvArgs a{};
    a.x = x->data, a.out = out->data;
    a.x_row = x->row_stride, a.out_row = out->row_stride;
    a.weight = h->weight, a.bias = h->weight + (size_t)h->width * h->channels;
    a.states = states, a.state_slots = state_slots;
    a.slots_in = slots_in, a.slots_out = slots_out, a.starts = starts;
    a.rows = rows, a.seqs = seqs, a.channels = h->channels;
    const uint32_t bytes = type_bytes(x->dtype), vector = 16 / bytes;
    const bool vectors = wide(x) && wide(out) && (uintptr_t)states % 16 == 0 && h->channels % vector == 0;
    const uint32_t per = CONV_LANES * (vectors ? vector : 4);
    a.columns = (h->channels + per - 1) / per;
    a.runs = row_blocks(CONV_RUN);
    const uint64_t blocks = (uint64_t)row_block_count(rows, seqs, a.runs.size) * a.columns;
    if (blocks > 1u << 25) return fail(RL_ERR_CAPACITY, "too many rows times channels in a call");
    with_type(x->dtype, [&](auto t) {
        with_width(h->width, [&](auto w) {
            using T = decltype(t);
            constexpr int W = decltype(w)::value;
            const bool act = h->activation == RL_CONV_SILU;
            if (vectors) launch_conv<T, W, true>(a, (uint32_t)blocks, act, static_cast<hipStream_t>(stream));
            else launch_conv<T, W, false>(a, (uint32_t)blocks, act, static_cast<hipStream_t>(stream));
        });
    });
    return launched("rl_conv_rows launch");
}

}  // extern "C"
