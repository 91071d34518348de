// C ABI of the token mixers (include/rl_mixers.h): handles, checks of arguments
// and launches. Kernels are in rotary.h, kv_cache.h, attend.h, delta.h and
// delta_chunks.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <new>
#include <string>

#include "attend.h"
#include "delta_launch.h"
#include "rl_runtime.h"

using namespace rl;

struct rl_rotary {
    int device = 0;
    rl_rotary_spec spec{};
    double magnitude = 1.0;
    double radians[ROTARY_MAX_PAIRS] = {};
    double *turns = nullptr; // device: revolutions a position
    ~rl_rotary() { (void)hipFree(turns); }
};

struct rl_kv_cache {
    int device = 0;
    CacheArgs args{};
    uint32_t format = 0;
    uint64_t bytes = 0;
    ~rl_kv_cache() {
        (void)hipFree(args.keys);
        (void)hipFree(args.values);
        (void)hipFree(args.key_steps);
        (void)hipFree(args.value_steps);
    }
};

struct rl_attention {
    int device = 0;
    uint32_t max_rows = 0, q_heads = 0, kv_heads = 0, dim = 0, max_len = 0;
    uint64_t slots = 0; // partial results of a row and head
    float *part_out = nullptr;
    float2 *part_sum = nullptr;
    uint32_t *part_count = nullptr, *arrived = nullptr;
    ~rl_attention() {
        (void)hipFree(part_out);
        (void)hipFree(part_sum);
        (void)hipFree(part_count);
        (void)hipFree(arrived);
    }
};

struct rl_delta {
    int device = 0;
    uint32_t max_rows = 0, max_seqs = 0, key_heads = 0, value_heads = 0, key_dim = 0, value_dim = 0;
    uint32_t chunks = 0; // that the workspace has room for
    DeltaWork work{};
    ~rl_delta() {
        (void)hipFree(work.kt);
        (void)hipFree(work.kf);
        (void)hipFree(work.qf);
        (void)hipFree(work.tm);
        (void)hipFree(work.pm);
        (void)hipFree(work.rows);
    }
};

namespace {

constexpr uint32_t MAX_ROWS = 1u << 23; // a workgroup of 256 threads a row stays below 2^32 threads

uint32_t type_bytes(uint32_t dtype) { return dtype == RL_F32 ? 4 : dtype == RL_F16 || dtype == RL_BF16 ? 2 : 1; }

// What is wrong with a tensor argument of a call of `rows` rows, or null.
const char *wrong(const rl_heads *h, uint32_t rows, bool written) {
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

bool wide(const rl_heads *h) {
    const uint64_t b = type_bytes(h->dtype);
    return (uintptr_t)h->data % 16 == 0 && h->row_stride * b % 16 == 0 && h->head_stride * b % 16 == 0;
}

RotaryArgs rotary_args(const rl_rotary *r, bool inverse) {
    RotaryArgs a{};
    if (!r) return a;
    a.turns = r->turns;
    a.pairs = r->spec.dims / 2;
    a.interleaved = r->spec.layout == RL_ROTARY_INTERLEAVED;
    a.magnitude = (float)r->magnitude;
    a.sign = inverse ? -1.0f : 1.0f;
    return a;
}

template <typename TI, typename TO, int V>
void launch_rotary(const RotaryArgs &r, const int64_t *positions, uint32_t rows, const RotaryTensor &a,
                   const RotaryTensor &b, hipStream_t s) {
    if (r.interleaved)
        hipLaunchKernelGGL((k_rotary<TI, TO, V == 1 ? 2 : V, true>), dim3(rows), dim3(ROTARY_THREADS), 0, s, r,
                           positions, a, b);
    else
        hipLaunchKernelGGL((k_rotary<TI, TO, V, false>), dim3(rows), dim3(ROTARY_THREADS), 0, s, r, positions, a, b);
}

// Calls f with a value of the element type.
template <typename F>
void with_type(uint32_t dtype, F f) {
    if (dtype == RL_F32) f(float{});
    else if (dtype == RL_F16) f(half_t{});
    else f(bhalf_t{});
}

CacheRows cache_rows(const rl_heads *k, const rl_heads *v, uint32_t rows) {
    CacheRows r{};
    r.keys = k->data, r.values = v->data;
    r.key_row = k->row_stride, r.key_head = k->head_stride;
    r.value_row = v->row_stride, r.value_head = v->head_stride;
    r.rows = rows;
    r.wide = wide(k) && wide(v);
    return r;
}

template <typename F>
void with_format(uint32_t format, F f) {
    if (format == RL_F16) f(std::integral_constant<int, RL_F16>{});
    else if (format == RL_BF16) f(std::integral_constant<int, RL_BF16>{});
    else if (format == RL_I8) f(std::integral_constant<int, RL_I8>{});
    else f(std::integral_constant<int, RL_F8>{});
}

// Lanes that hold a vector of `dim` values, eight each.
template <typename F>
void with_group(uint32_t dim, F f) {
    if (dim <= 64) f(std::integral_constant<int, 8>{});
    else if (dim <= 128) f(std::integral_constant<int, 16>{});
    else f(std::integral_constant<int, 32>{});
}

int check_cache_rows(const rl_kv_cache *c, const rl_heads *k, const rl_heads *v, const int64_t *slots, uint32_t rows,
                     bool written) {
    if (!c) return fail(RL_ERR_ARGUMENT, "cache is null");
    CHECK_HEADS(k, "keys", written);
    CHECK_HEADS(v, "values", written);
    if (k->dtype != v->dtype) return fail(RL_ERR_ARGUMENT, "keys and values differ in type");
    for (const rl_heads *h : {k, v})
        if (h->heads != c->args.heads || h->dim != c->args.dim)
            return fail(RL_ERR_ARGUMENT, "keys and values must have the cache's heads and dim");
    if (rows && !slots) return fail(RL_ERR_ARGUMENT, "slots must be a device pointer");
    if (rows > MAX_ROWS) return fail(RL_ERR_CAPACITY, "more than 2^23 rows in a call");
    return RL_OK;
}

// Parts of a row's length are at most ATTEND_LONG tokens, so that a batch of very
// different lengths is shared out evenly, and otherwise as many as give each CU
// the workgroups it holds at a time, each a tile of 32 tokens a wave or more. 64
// int8 sequences of 128 to 8192 tokens: 70.2 us with 768 or 1024, 71.0 with 1536,
// 71.7 with 2048, 83 with 4096; 1536 joins less where lengths are alike. One
// sequence of 131071 tokens took 114 us with the limit, 97 without.
constexpr uint32_t ATTEND_LONG = 1536, CUS = 256;

uint32_t attend_tiles(uint64_t tokens) { return (uint32_t)((tokens + ATTEND_TILE - 1) / ATTEND_TILE) + 1; }

// Partial results that a handle has room for at most, 0.5 GB of them for heads of 128. Calls of more rows times heads than
// this holds parts for have row blocks enough to fill the device. Without a limit 8192 rows of 32 heads and lengths up to
// 131072 took 11.7 GB, a million tokens 35.
constexpr uint64_t ATTEND_ROOM = 1u << 20;

// Parts that lengths up to `tiles` need at the least; one sequence has no others to wait for.
uint32_t attend_least_parts(uint32_t tiles, uint32_t seqs) {
    if (seqs == 1) return 1;
    const uint32_t n = (tiles + ATTEND_LONG / ATTEND_TILE - 1) / (ATTEND_LONG / ATTEND_TILE);
    return std::min(n, ATTEND_MAX_PARTS);
}

// Rows of a sequence from which chunks are faster than one token after the other (us, steps / chunks; 32 heads of 128 x
// 128). While every workgroup of the chunks has a CU to itself they cost the same for any rows up to 64: one bf16
// sequence of 12 rows 15.4 / 16.1, of 16 19.3 / 16.1; f32, more products, 16 rows 17.0 / 22.5, 24 rows 23.2 / 22.5. Beyond
// that they wait for each other: 16 sequences of 16 rows 54.6 / 79, of 24 76.2 / 78.7, of 32 98.7 / 78.3.
constexpr uint32_t DELTA_CHUNKED = 13, DELTA_CHUNKED_WIDE = 20, DELTA_CHUNKED_MANY = 25;

int launched(const char *what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? RL_OK : hip_fail(e, what);
}

}  // namespace

extern "C" {

int rl_rotary_create(int device, const rl_rotary_spec *spec, rl_rotary **out) {
    if (!out) return fail(RL_ERR_ARGUMENT, "out is null");
    *out = nullptr;
    if (!spec) return fail(RL_ERR_ARGUMENT, "spec is null");
    const uint32_t d = spec->dims;
    if (d < 2 || d % 2 || d > 2 * ROTARY_MAX_PAIRS) return fail(RL_ERR_ARGUMENT, "dims must be even, from 2 to 512");
    if (spec->layout > RL_ROTARY_INTERLEAVED) return fail(RL_ERR_ARGUMENT, "unknown rotary layout");
    if (spec->scaling > RL_ROTARY_YARN) return fail(RL_ERR_ARGUMENT, "unknown rotary scaling");
    if (!(spec->base > 1.0) || !std::isfinite(spec->base)) return fail(RL_ERR_ARGUMENT, "base must be above 1");
    if (spec->scaling != RL_ROTARY_PLAIN && (!(spec->factor >= 1.0) || !std::isfinite(spec->factor)))
        return fail(RL_ERR_ARGUMENT, "factor must be at least 1");
    if (spec->scaling == RL_ROTARY_NTK && d == 2) return fail(RL_ERR_ARGUMENT, "ntk scaling needs more than 2 dims");
    if (!(spec->magnitude >= 0.0) || !std::isfinite(spec->magnitude))
        return fail(RL_ERR_ARGUMENT, "magnitude must not be negative");
    const double fast = spec->beta_fast == 0.0 ? 32.0 : spec->beta_fast;
    const double slow = spec->beta_slow == 0.0 ? 1.0 : spec->beta_slow;
    if (spec->scaling == RL_ROTARY_YARN) {
        if (spec->original == 0) return fail(RL_ERR_ARGUMENT, "yarn scaling needs the original context");
        if (!(slow > 0.0) || !(fast >= slow) || !std::isfinite(fast))
            return fail(RL_ERR_ARGUMENT, "beta_fast must be at least beta_slow, both positive");
    }
    DeviceGuard guard(device);
    if (!guard.ok) return fail(RL_ERR_DEVICE, "cannot select device " + std::to_string(device));
    auto *r = new (std::nothrow) rl_rotary();
    if (!r) return fail(RL_ERR_CAPACITY, "out of host memory");
    r->device = device;
    r->spec = *spec;
    constexpr double TWO_PI = 6.283185307179586476925;
    double base = spec->base;
    if (spec->scaling == RL_ROTARY_NTK) base *= std::pow(spec->factor, (double)d / (d - 2));
    // The pair whose angle takes `turns` revolutions over the original context.
    auto place = [&](double turns) {
        return d * std::log(spec->original / (turns * TWO_PI)) / (2.0 * std::log(spec->base));
    };
    double low = 0.0, high = 0.0;
    if (spec->scaling == RL_ROTARY_YARN) {
        low = std::max(std::floor(place(fast)), 0.0);
        high = std::min(std::ceil(place(slow)), (double)d - 1.0);
    }
    double turns[ROTARY_MAX_PAIRS] = {};
    for (uint32_t i = 0; i < d / 2; i++) {
        double f = std::pow(base, -2.0 * i / d);
        if (spec->scaling == RL_ROTARY_LINEAR) f /= spec->factor;
        if (spec->scaling == RL_ROTARY_YARN) {
            const double ramp = std::min(std::max((i - low) / std::max(high - low, 0.001), 0.0), 1.0);
            f = f * (1.0 - ramp) + f / spec->factor * ramp;
        }
        r->radians[i] = f;
        turns[i] = f / TWO_PI;
    }
    r->magnitude = spec->magnitude != 0.0 ? spec->magnitude
                   : spec->scaling == RL_ROTARY_YARN ? 0.1 * std::log(spec->factor) + 1.0
                                                     : 1.0;
    hipError_t e = hipMalloc(&r->turns, sizeof turns);
    if (e == hipSuccess) e = hipMemcpy(r->turns, turns, sizeof turns, hipMemcpyHostToDevice);
    if (e != hipSuccess) {
        delete r;
        return hip_fail(e, "rl_rotary_create");
    }
    *out = r;
    return RL_OK;
}

void rl_rotary_destroy(rl_rotary *rotary) {
    if (!rotary) return;
    DeviceGuard guard(rotary->device);
    delete rotary;
}

int rl_rotary_frequencies(const rl_rotary *r, double *radians, double *magnitude) {
    if (!r) return fail(RL_ERR_ARGUMENT, "rotary is null");
    if (radians) std::copy(r->radians, r->radians + r->spec.dims / 2, radians);
    if (magnitude) *magnitude = r->magnitude;
    return RL_OK;
}

int rl_rotary_rows(rl_rotary *r, const int64_t *positions, uint32_t rows, const rl_heads *in, const rl_heads *out,
                   uint32_t tensors, int inverse, void *stream) {
    if (!r) return fail(RL_ERR_ARGUMENT, "rotary is null");
    if (!in || !out || tensors < 1 || tensors > 2) return fail(RL_ERR_ARGUMENT, "one or two tensors are turned");
    bool all_wide = true;
    for (uint32_t i = 0; i < tensors; i++) {
        CHECK_HEADS(in + i, "in", false);
        CHECK_HEADS(out + i, "out", true);
        if (in[i].heads != out[i].heads || in[i].dim != out[i].dim)
            return fail(RL_ERR_ARGUMENT, "in and out differ in shape");
        if (in[i].dim < r->spec.dims) return fail(RL_ERR_ARGUMENT, "dim below the turned values");
        if (in[i].dtype != in[0].dtype || out[i].dtype != out[0].dtype)
            return fail(RL_ERR_ARGUMENT, "the tensors of a call have one type");
        if (in[i].data == out[i].data && (in[i].dtype != out[i].dtype || in[i].row_stride != out[i].row_stride ||
                                          in[i].head_stride != out[i].head_stride))
            return fail(RL_ERR_ARGUMENT, "in place needs the same type and strides");
        if ((uint64_t)in[i].heads * in[i].dim > 1u << 24) return fail(RL_ERR_CAPACITY, "more than 2^24 values a row");
        all_wide &= wide(in + i) && wide(out + i);
    }
    if (rows == 0) return RL_OK;
    if (!positions) return fail(RL_ERR_ARGUMENT, "positions must be a device pointer");
    if (rows > MAX_ROWS) return fail(RL_ERR_CAPACITY, "more than 2^23 rows in a call");
    DeviceGuard guard(r->device);
    if (!guard.ok) return fail(RL_ERR_DEVICE, "cannot select the handle's device");
    const RotaryArgs args = rotary_args(r, inverse != 0);
    // Eight values at a time (four if either side is f32) where the turned part splits into such units.
    const uint32_t most = in->dtype == RL_F32 || out->dtype == RL_F32 ? 4 : 8;
    const uint32_t part = args.interleaved ? 2 * args.pairs : args.pairs;
    const uint32_t v = all_wide && part % most == 0 ? most : args.interleaved ? 2 : 1;
    RotaryTensor t[2] = {};
    for (uint32_t i = 0; i < tensors; i++) {
        t[i].in = in[i].data, t[i].out = out[i].data;
        t[i].in_row = in[i].row_stride, t[i].in_head = in[i].head_stride;
        t[i].out_row = out[i].row_stride, t[i].out_head = out[i].head_stride;
        t[i].heads = in[i].heads, t[i].dim = in[i].dim;
        t[i].units = part / v + (in[i].dim - 2 * args.pairs + v - 1) / v;
        t[i].wide = v >= 4;
    }
    with_type(in->dtype, [&](auto ti) {
        with_type(out->dtype, [&](auto to) {
            using TI = decltype(ti);
            using TO = decltype(to);
            constexpr int MOST = sizeof(TI) == 4 || sizeof(TO) == 4 ? 4 : 8;
            if (v == MOST)
                launch_rotary<TI, TO, MOST>(args, positions, rows, t[0], t[1], static_cast<hipStream_t>(stream));
            else
                launch_rotary<TI, TO, 1>(args, positions, rows, t[0], t[1], static_cast<hipStream_t>(stream));
        });
    });
    return launched("rl_rotary_rows launch");
}

int rl_kv_cache_create(int device, uint32_t pages, uint32_t page, uint32_t kv_heads, uint32_t dim, uint32_t format,
                       rl_kv_cache **out) {
    if (!out) return fail(RL_ERR_ARGUMENT, "out is null");
    *out = nullptr;
    if (pages == 0 || page == 0 || kv_heads == 0) return fail(RL_ERR_ARGUMENT, "pages, page and kv_heads must be positive");
    if (dim < 16 || dim > 256 || dim % 16) return fail(RL_ERR_ARGUMENT, "dim must be a multiple of 16, from 16 to 256");
    if (format < RL_F16 || format > RL_F8) return fail(RL_ERR_ARGUMENT, "unknown cache format");
    const uint64_t slots = (uint64_t)pages * page;
    if (slots > 1ull << 32 || kv_heads > 1u << 16) return fail(RL_ERR_CAPACITY, "the cache is too large");
    DeviceGuard guard(device);
    if (!guard.ok) return fail(RL_ERR_DEVICE, "cannot select device " + std::to_string(device));
    auto *c = new (std::nothrow) rl_kv_cache();
    if (!c) return fail(RL_ERR_CAPACITY, "out of host memory");
    c->device = device;
    c->format = format;
    c->args.slots = slots;
    c->args.page = page, c->args.heads = kv_heads, c->args.dim = dim;
    c->args.page_inv = inverse_of(page), c->args.vectors_inv = inverse_of(2 * kv_heads);
    const uint64_t codes = slots * kv_heads * dim * type_bytes(format), steps = slots * kv_heads * sizeof(float);
    hipError_t e = hipMalloc(&c->args.keys, codes);
    if (e == hipSuccess) e = hipMalloc(&c->args.values, codes);
    if (e == hipSuccess) e = hipMemset(c->args.keys, 0, codes);
    if (e == hipSuccess) e = hipMemset(c->args.values, 0, codes);
    c->bytes = 2 * codes;
    if (format == RL_I8 || format == RL_F8) {
        if (e == hipSuccess) e = hipMalloc(&c->args.key_steps, steps);
        if (e == hipSuccess) e = hipMalloc(&c->args.value_steps, steps);
        if (e == hipSuccess) e = hipMemset(c->args.key_steps, 0, steps);
        if (e == hipSuccess) e = hipMemset(c->args.value_steps, 0, steps);
        c->bytes += 2 * steps;
    }
    if (e == hipSuccess) e = hipDeviceSynchronize();
    if (e != hipSuccess) {
        delete c;
        return hip_fail(e, "rl_kv_cache_create");
    }
    *out = c;
    return RL_OK;
}

void rl_kv_cache_destroy(rl_kv_cache *cache) {
    if (!cache) return;
    DeviceGuard guard(cache->device);
    delete cache;
}

uint64_t rl_kv_cache_bytes(const rl_kv_cache *cache) { return cache ? cache->bytes : 0; }

int rl_kv_cache_write(rl_kv_cache *c, const rl_heads *keys, const rl_heads *values, const int64_t *slots,
                      uint32_t rows, const rl_rotary *rotary, const int64_t *positions, void *stream) {
    if (const int rc = check_cache_rows(c, keys, values, slots, rows, false)) return rc;
    if (rotary && rotary->spec.dims > c->args.dim) return fail(RL_ERR_ARGUMENT, "dim below the turned values");
    if (rotary && rotary->device != c->device) return fail(RL_ERR_ARGUMENT, "the rotary handle is on another device");
    if (rotary && rows && !positions) return fail(RL_ERR_ARGUMENT, "positions must be a device pointer");
    if (rows == 0) return RL_OK;
    DeviceGuard guard(c->device);
    if (!guard.ok) return fail(RL_ERR_DEVICE, "cannot select the cache's device");
    const CacheRows in = cache_rows(keys, values, rows);
    const RotaryArgs r = rotary_args(rotary, false);
    with_type(keys->dtype, [&](auto t) {
        with_format(c->format, [&](auto f) {
            with_group(c->args.dim, [&](auto g) {
                constexpr int G = decltype(g)::value;
                // As many rows as give each group of lanes the vectors it loads ahead where the workgroups are four a CU or
                // more with one; with fewer the shorter chain counts (8 heads of 128 to int8, us, ahead / one: 64 rows
                // 3.7 / 3.0, 512 3.9 / 3.5, 1024 4.4 / 4.4, 2048 5.9 / 6.5, 4096 9.1 / 10.1).
                constexpr uint32_t GROUPS = CACHE_THREADS / G;
                const bool many = (uint64_t)rows * 2 * c->args.heads / GROUPS >= 4 * CUS;
                const uint32_t vectors = GROUPS * (many ? CACHE_AHEAD : 1);
                const uint32_t per = std::min(std::max(vectors / (2 * c->args.heads), 1u), CACHE_MAX_ROWS);
                hipLaunchKernelGGL((k_cache_write<decltype(t), decltype(f)::value, G>), dim3((rows + per - 1) / per),
                                   dim3(CACHE_THREADS), 0, static_cast<hipStream_t>(stream), c->args, in, slots, per, r,
                                   positions);
            });
        });
    });
    return launched("rl_kv_cache_write launch");
}

int rl_kv_cache_read(rl_kv_cache *c, const int64_t *slots, uint32_t rows, const rl_heads *keys,
                     const rl_heads *values, void *stream) {
    if (const int rc = check_cache_rows(c, keys, values, slots, rows, true)) return rc;
    if (rows == 0) return RL_OK;
    DeviceGuard guard(c->device);
    if (!guard.ok) return fail(RL_ERR_DEVICE, "cannot select the cache's device");
    const CacheRows out = cache_rows(keys, values, rows);
    uint64_t blocks = 0;
    with_group(c->args.dim, [&](auto g) {
        constexpr uint32_t PER = CACHE_THREADS / decltype(g)::value;
        blocks = ((uint64_t)rows * 2 * c->args.heads + PER - 1) / PER;
    });
    if (blocks > MAX_ROWS) return fail(RL_ERR_CAPACITY, "too many heads in a call");
    with_type(keys->dtype, [&](auto t) {
        with_format(c->format, [&](auto f) {
            with_group(c->args.dim, [&](auto g) {
                hipLaunchKernelGGL((k_cache_read<decltype(t), decltype(f)::value, decltype(g)::value>),
                                   dim3((uint32_t)blocks), dim3(CACHE_THREADS), 0, static_cast<hipStream_t>(stream),
                                   c->args, out, slots);
            });
        });
    });
    return launched("rl_kv_cache_read launch");
}

int rl_attention_create(int device, uint32_t max_rows, uint32_t q_heads, uint32_t kv_heads, uint32_t dim,
                        uint32_t max_len, rl_attention **out) {
    if (!out) return fail(RL_ERR_ARGUMENT, "out is null");
    *out = nullptr;
    if (max_rows == 0 || max_len == 0 || kv_heads == 0 || q_heads == 0 || q_heads % kv_heads)
        return fail(RL_ERR_ARGUMENT, "max_rows and max_len must be positive, q_heads a multiple of kv_heads");
    if (dim < 16 || dim > 256 || dim % 16) return fail(RL_ERR_ARGUMENT, "dim must be a multiple of 16, from 16 to 256");
    if ((uint64_t)max_rows * q_heads > MAX_ROWS || max_len > 0x7FFFFFFFu)
        return fail(RL_ERR_CAPACITY, "max_rows * q_heads above 2^23 or max_len above 2^31 - 1");
    DeviceGuard guard(device);
    if (!guard.ok) return fail(RL_ERR_DEVICE, "cannot select device " + std::to_string(device));
    auto *a = new (std::nothrow) rl_attention();
    if (!a) return fail(RL_ERR_CAPACITY, "out of host memory");
    a->device = device;
    a->max_rows = max_rows, a->q_heads = q_heads, a->kv_heads = kv_heads, a->dim = dim, a->max_len = max_len;
    // Room for the least parts of every row within the limit, and for as many workgroups of 32 rows as the device holds.
    const uint64_t heads = (uint64_t)max_rows * q_heads;
    a->slots = std::max<uint64_t>(std::min(heads * attend_least_parts(attend_tiles(max_len), 2), ATTEND_ROOM), CUS * 3 * 32);
    hipError_t e = hipMalloc(&a->part_out, a->slots * attend_dim(dim) * sizeof(float));
    if (e == hipSuccess) e = hipMalloc(&a->part_sum, a->slots * sizeof(float2));
    if (e == hipSuccess) e = hipMalloc(&a->part_count, heads * sizeof(uint32_t));
    if (e == hipSuccess) e = hipMalloc(&a->arrived, heads * sizeof(uint32_t));
    if (e == hipSuccess) e = hipMemset(a->part_count, 0, heads * sizeof(uint32_t));
    if (e == hipSuccess) e = hipMemset(a->arrived, 0, heads * sizeof(uint32_t));
    if (e == hipSuccess) e = hipDeviceSynchronize();
    if (e != hipSuccess) {
        delete a;
        return hip_fail(e, "rl_attention_create");
    }
    *out = a;
    return RL_OK;
}

void rl_attention_destroy(rl_attention *attention) {
    if (!attention) return;
    DeviceGuard guard(attention->device);
    delete attention;
}

int rl_attention_rows(rl_attention *h, const rl_kv_cache *cache, const rl_heads *q, const rl_heads *out, float *lse,
                      uint32_t rows, const int32_t *starts, const int32_t *lens, uint32_t seqs, const int32_t *pages,
                      uint32_t table_width, float scale, uint32_t window, uint32_t most_rows, uint32_t max_len,
                      void *stream) {
    if (!h) return fail(RL_ERR_ARGUMENT, "attention is null");
    if (!cache) return fail(RL_ERR_ARGUMENT, "cache is null");
    CHECK_HEADS(q, "q", false);
    CHECK_HEADS(out, "out", true);
    if (cache->device != h->device) return fail(RL_ERR_ARGUMENT, "the cache is on another device");
    if (cache->args.heads != h->kv_heads || cache->args.dim != h->dim)
        return fail(RL_ERR_ARGUMENT, "the cache has other heads or another dim than the handle");
    if (q->heads != h->q_heads || q->dim != h->dim || out->heads != h->q_heads || out->dim != h->dim)
        return fail(RL_ERR_ARGUMENT, "q and out must have the handle's heads and dim");
    if (q->dtype != out->dtype) return fail(RL_ERR_ARGUMENT, "q and out differ in type");
    if ((cache->format == RL_F16 && q->dtype == RL_BF16) || (cache->format == RL_BF16 && q->dtype == RL_F16))
        return fail(RL_ERR_ARGUMENT, "an f16 cache takes f16 or f32 queries, a bf16 cache bf16 or f32");
    if (rows > h->max_rows) return fail(RL_ERR_CAPACITY, "rows above the handle's max_rows");
    if (max_len > h->max_len) return fail(RL_ERR_CAPACITY, "max_len above the handle's");
    if (rows == 0) return RL_OK;
    if (!lens || !pages || table_width == 0) return fail(RL_ERR_ARGUMENT, "lens and pages must be device pointers");
    if (seqs == 0 || (!starts && seqs != rows)) return fail(RL_ERR_ARGUMENT, "without starts there is one row a sequence");
    if (window > 0x7FFFFFFFu) window = 0; // no length is above it
    DeviceGuard guard(h->device);
    if (!guard.ok) return fail(RL_ERR_DEVICE, "cannot select the handle's device");
    AttendArgs a{};
    a.cache = cache->args;
    a.q = q->data, a.out = out->data, a.lse = lse;
    a.q_row = q->row_stride, a.q_head = q->head_stride;
    a.out_row = out->row_stride, a.out_head = out->head_stride;
    a.starts = starts, a.lens = lens, a.pages = pages;
    a.rows = rows, a.seqs = seqs, a.q_heads = h->q_heads, a.table_width = table_width, a.window = window;
    a.most_rows = !starts ? 1 : most_rows ? std::min(most_rows, rows) : rows;
    a.max_len = max_len ? max_len : h->max_len;
    a.scale = scale;
    a.group = h->q_heads / h->kv_heads;
    a.wide = wide(q) && wide(out);
    a.part_out = h->part_out, a.part_sum = h->part_sum, a.part_count = h->part_count, a.arrived = h->arrived;
    const uint64_t expanded = (uint64_t)a.most_rows * a.group;
    const bool two = attend_two(cache->format, h->dim, (expanded + 15) / 16, (uint64_t)seqs * h->kv_heads);
    const uint32_t block_rows = two ? 32 : 16;
    // A grid of the longest sequence's row blocks for every sequence, or of the sum of all. The second asks each workgroup to
    // find its sequence, and is taken where it is less than half as large; the first can pass what a launch takes. 64
    // sequences of 2048 tokens, 32 / 8 heads of 128 bf16, us, first / second: all with 64 rows 844 / 899, 21 of them (the
    // others one) 509 / 374, one 361 / 133; eight with 9 rows 115 / 121.
    const uint64_t longest = (expanded + block_rows - 1) / block_rows, sum = (uint64_t)rows * a.group / block_rows + seqs;
    a.packed = sum * 2 < longest * seqs;
    a.blocks = (uint32_t)(a.packed ? sum : longest);
    const uint64_t columns = (uint64_t)(a.packed ? 1 : seqs) * h->kv_heads * a.blocks;
    const uint64_t seen = window ? std::min<uint64_t>(a.max_len, (uint64_t)window + a.most_rows - 1) : a.max_len;
    const uint32_t tiles = attend_tiles(seen);
    const uint64_t room = std::min<uint64_t>(h->slots / ((uint64_t)rows * h->q_heads), ATTEND_MAX_PARTS);
    const uint64_t held = CUS * attend_resident(type_bytes(q->dtype), cache->format, h->dim, two ? 2 : 1);
    uint64_t parts = std::max<uint64_t>(held / columns, attend_least_parts(tiles, seqs));
    parts = std::max<uint64_t>(std::min(parts, room), 1);
    a.part_tiles = (uint32_t)((tiles + parts - 1) / parts);
    a.part_tiles = (a.part_tiles + ATTEND_WAVES - 1) / ATTEND_WAVES * ATTEND_WAVES;
    a.parts = (tiles + a.part_tiles - 1) / a.part_tiles;
    a.joins = a.parts <= ATTEND_FEW;
    a.group_inv = inverse_of(a.group), a.blocks_inv = inverse_of(a.blocks), a.heads_inv = inverse_of(h->kv_heads);
    a.columns_inv = inverse_of(seqs * h->kv_heads), a.tiles_inv = inverse_of(a.part_tiles);
    // Jobs (sequence, head and part) in eights, the row blocks of each eight together; or eight runs of row blocks at a time.
    constexpr uint64_t RUNS = 8 * ATTEND_RUN;
    const uint64_t groups = a.packed ? (columns * a.parts + RUNS - 1) / RUNS * RUNS
                                     : ((uint64_t)seqs * h->kv_heads * a.parts + 7) / 8 * 8 * a.blocks;
    if (groups > 2 * MAX_ROWS - 1) return fail(RL_ERR_CAPACITY, "too many sequences times row blocks in a call");
    with_type(q->dtype, [&](auto t) {
        launch_attend<decltype(t)>(a, cache->format, two, (uint32_t)groups, static_cast<hipStream_t>(stream));
    });
    return launched("rl_attention_rows launch");
}

int rl_delta_create(int device, uint32_t max_rows, uint32_t max_seqs, uint32_t key_heads, uint32_t value_heads,
                    uint32_t key_dim, uint32_t value_dim, rl_delta **out) {
    if (!out) return fail(RL_ERR_ARGUMENT, "out is null");
    *out = nullptr;
    if (max_rows == 0 || max_seqs == 0 || key_heads == 0 || value_heads == 0 || value_heads % key_heads)
        return fail(RL_ERR_ARGUMENT, "max_rows and max_seqs must be positive, value_heads a multiple of key_heads");
    for (uint32_t d : {key_dim, value_dim})
        if (d < 16 || d > 256 || d % 16)
            return fail(RL_ERR_ARGUMENT, "key_dim and value_dim must be multiples of 16, from 16 to 256");
    if (max_rows > MAX_ROWS || (uint64_t)max_seqs * value_heads > MAX_ROWS)
        return fail(RL_ERR_CAPACITY, "max_rows or max_seqs * value_heads above 2^23");
    DeviceGuard guard(device);
    if (!guard.ok) return fail(RL_ERR_DEVICE, "cannot select device " + std::to_string(device));
    auto *d = new (std::nothrow) rl_delta();
    if (!d) return fail(RL_ERR_CAPACITY, "out of host memory");
    d->device = device;
    d->max_rows = max_rows, d->max_seqs = max_seqs, d->key_heads = key_heads, d->value_heads = value_heads;
    d->key_dim = key_dim, d->value_dim = value_dim;
    if (max_rows >= DELTA_CHUNKED) {
        // Room for a prompt of every row, and for as many sequences as have 16 rows each on average, in f32.
        d->chunks = max_rows / CHUNK + std::min(max_seqs, max_rows / 16 + 1);
        const uint64_t heads = (uint64_t)d->chunks * value_heads;
        if (heads > MAX_ROWS) {
            delete d;
            return fail(RL_ERR_CAPACITY, "chunks of max_rows times value_heads above 2^23");
        }
        const uint64_t keys = (uint64_t)d->chunks * key_heads * key_size(delta_dim(key_dim)) * sizeof(float);
        hipError_t e = hipMalloc(&d->work.kt, keys);
        if (e == hipSuccess) e = hipMalloc(&d->work.kf, keys);
        if (e == hipSuccess) e = hipMalloc(&d->work.qf, keys);
        if (e == hipSuccess) e = hipMalloc(&d->work.tm, heads * 3 * SQUARE * sizeof(bhalf_t));
        if (e == hipSuccess) e = hipMalloc(&d->work.pm, heads * SQUARE * sizeof(float));
        if (e == hipSuccess) e = hipMalloc(&d->work.rows, heads * 4 * CHUNK * sizeof(float));
        if (e != hipSuccess) {
            delete d;
            return hip_fail(e, "rl_delta_create");
        }
    }
    *out = d;
    return RL_OK;
}

void rl_delta_destroy(rl_delta *delta) {
    if (!delta) return;
    DeviceGuard guard(delta->device);
    delete delta;
}

int rl_delta_rows(rl_delta *h, const rl_heads *q, const rl_heads *k, const rl_heads *v, const rl_heads *out,
                  const float *g, uint64_t g_stride, const float *beta, uint64_t beta_stride, float *states,
                  uint64_t state_slots, const int32_t *slots_in, const int32_t *slots_out, const int32_t *starts,
                  uint32_t rows, uint32_t seqs, float scale, float norm_eps, uint32_t most_rows, void *stream) {
    if (!h) return fail(RL_ERR_ARGUMENT, "delta is null");
    CHECK_HEADS(q, "q", false);
    CHECK_HEADS(k, "k", false);
    CHECK_HEADS(v, "v", false);
    CHECK_HEADS(out, "out", true);
    for (const rl_heads *x : {q, k})
        if (x->heads != h->key_heads || x->dim != h->key_dim)
            return fail(RL_ERR_ARGUMENT, "q and k must have the handle's key heads and key_dim");
    for (const rl_heads *x : {v, out})
        if (x->heads != h->value_heads || x->dim != h->value_dim)
            return fail(RL_ERR_ARGUMENT, "v and out must have the handle's value heads and value_dim");
    for (const rl_heads *x : {k, v, out})
        if (x->dtype != q->dtype) return fail(RL_ERR_ARGUMENT, "q, k, v and out have one type");
    if (rows > h->max_rows || seqs > h->max_seqs) return fail(RL_ERR_CAPACITY, "rows or seqs above the handle's");
    if (seqs == 0) return rows == 0 ? RL_OK : fail(RL_ERR_ARGUMENT, "rows without sequences");
    if ((rows && (!g || !beta)) || !states || !slots_in || !slots_out)
        return fail(RL_ERR_ARGUMENT, "g, beta, states and slots must be device pointers");
    if ((uintptr_t)states % 16) return fail(RL_ERR_ARGUMENT, "states must be aligned to 16 bytes");
    if (!starts && rows != seqs) return fail(RL_ERR_ARGUMENT, "without starts there is one row a sequence");
    if (std::isnan(scale) || std::isnan(norm_eps)) return fail(RL_ERR_ARGUMENT, "scale or norm_eps is NaN");
    DeviceGuard guard(h->device);
    if (!guard.ok) return fail(RL_ERR_DEVICE, "cannot select the handle's device");
    DeltaArgs a{};
    a.q = q->data, a.k = k->data, a.v = v->data, a.out = out->data;
    a.q_row = q->row_stride, a.q_head = q->head_stride, a.k_row = k->row_stride, a.k_head = k->head_stride;
    a.v_row = v->row_stride, a.v_head = v->head_stride, a.out_row = out->row_stride, a.out_head = out->head_stride;
    a.g = g, a.beta = beta, a.g_row = g_stride, a.beta_row = beta_stride;
    a.states = states, a.state_slots = state_slots, a.slots_in = slots_in, a.slots_out = slots_out, a.starts = starts;
    a.rows = rows, a.seqs = seqs, a.key_heads = h->key_heads, a.value_heads = h->value_heads;
    a.key_dim = h->key_dim, a.value_dim = h->value_dim;
    a.scale = scale, a.eps = norm_eps;
    a.wide = wide(q) && wide(k) && wide(v) && wide(out);
    // Chunks where some sequence has the rows for them, the workspace holds all and one launch too (below 2^32 threads).
    const uint32_t most = !starts ? 1 : most_rows ? std::min(most_rows, rows) : rows;
    const bool alone = (uint64_t)seqs * h->value_heads * (h->value_dim / 16) <= CUS;
    const uint32_t least = !alone ? DELTA_CHUNKED_MANY : q->dtype == RL_BF16 ? DELTA_CHUNKED : DELTA_CHUNKED_WIDE;
    const uint64_t groups = delta_groups(a);
    const bool chunked = most >= least && rows / CHUNK + seqs <= h->chunks && groups * DELTA_CHUNK_THREADS < 1ull << 32;
    with_type(q->dtype, [&](auto t) {
        if (chunked) launch_delta_chunks<decltype(t)>(a, h->work, static_cast<hipStream_t>(stream));
        else launch_delta_steps<decltype(t)>(a, static_cast<hipStream_t>(stream));
    });
    return launched("rl_delta_rows launch");
}

}  // extern "C"
