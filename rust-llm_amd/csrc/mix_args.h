// Checks of the token mixers' arguments and their dispatch by element type, for the
// units that hold the C ABI (include/rl_mixers.h).
#pragma once
#include <string>

#include "mix_types.h"
#include "rl_runtime.h"

namespace rl {

constexpr uint32_t MAX_ROWS = 1u << 23; // a workgroup of 256 threads a row stays below 2^32 threads

inline uint32_t type_bytes(uint32_t dtype) { return dtype == RL_F32 ? 4 : dtype == RL_F16 || dtype == RL_BF16 ? 2 : 1; }

// What is wrong with a tensor argument of a call of `rows` rows, or null.
inline const char *wrong(const rl_heads *h, uint32_t rows, bool written) {
    if (!h) return "is null";
    if (!h->data && rows) return "has no data";
    if (h->dtype > RL_BF16) return "must be f32, f16 or bf16";
    if (h->heads == 0 || h->dim == 0) return "has no heads or no values";
    if ((uintptr_t)h->data % type_bytes(h->dtype)) return "is not aligned to its type";
    if (written && h->heads > 1 && h->head_stride < h->dim) return "is written with overlapping heads";
    if (written && rows > 1 && h->row_stride < h->dim) return "is written with overlapping rows";
    return nullptr;
}

#define CHECK_HEADS(h, name, written) /* of a call's `rows` */                                                     \
    do {                                                                                           \
        if (const char *w = wrong(h, rows, written)) return fail(RL_ERR_ARGUMENT, std::string(name) + " " + w); \
    } while (0)

inline bool wide(const rl_heads *h) {
    const uint64_t b = type_bytes(h->dtype);
    return (uintptr_t)h->data % 16 == 0 && h->row_stride * b % 16 == 0 && h->head_stride * b % 16 == 0;
}

// Calls f with a value of the element type.
template <typename F>
void with_type(uint32_t dtype, F f) {
    if (dtype == RL_F32) f(float{});
    else if (dtype == RL_F16) f(half_t{});
    else f(bhalf_t{});
}

inline int launched(const char *what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? RL_OK : hip_fail(e, what);
}

}  // namespace rl
