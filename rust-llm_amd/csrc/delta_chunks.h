// The gated delta rule over many tokens (include/rl_mixers.h): chunks of 64
// tokens on the matrix cores.
//
// With c_i the sum of g over a chunk's tokens up to i and S the state before the
// chunk, the corrected values u of its tokens solve a unit lower triangular system,
//   (1 + L) U = B (V - diag(e^c) K S),  L_ij = beta_i (k_i . k_j) e^(c_i - c_j), j < i
// and, with e^c_n the decay of the whole chunk,
//   out = diag(e^c) Q S + P U,          P_ij = (q_i . k_j) e^(c_i - c_j), j <= i
//   S  <- e^c_n S + K^T diag(e^(c_n - c)) U
// k_delta_prepare forms T = (1 + L)^-1 B and P for every chunk at once.
// k_delta_chunks then goes through a sequence's chunks, a workgroup for 16 columns
// of a head's state: the columns do not depend on each other.
//
// Every product is bf16 on the matrix cores with f32 sums. What has more than
// bf16's 8 bits is split into parts that add up to it: three for the state, T, the
// corrected values and f32 queries and keys (24 bits), two for f16 ones. Products
// of split operands leave out what lies below 2^-24 of them (lo lo, mid lo). Two
// parts would do for 16-bit outputs, but the state is an f32 result that goes from
// chunk to chunk: with two it was 9e-6 off f64 at the end of 700 tokens, with three
// it is as near as f32 arithmetic. Where the output is bf16, what only the output
// takes (P, and there the state and the corrected values) has two parts, 16 bits:
// they add less than a thousandth to the error of its rounding. With P in one part
// that error was 1.38 times as large, and 8192 tokens took 288 us instead of 305.
// Decays are differences of f64 sums, so that a token after a strong decay is as
// exact as one before.
#pragma once
#include "delta.h"

namespace rl {

constexpr uint32_t CHUNK = 64;

// Operands of the chunks, zeros where a chunk or a head ends early, as fragments: for each of 64 lanes eight values, row
// lane % 16 of a 16-row tile, columns 8 (lane / 16) on of a step of 32. K and
// Q too: read where they are, a token's 4 KB or so from the next, all rows of a
// head come from one channel of the L2 (3.1 us a chunk; now 1.9).
struct DeltaWork {
    void *kt;    // [chunk][key head][DK/16 tiles][2 steps]: K^T in the call's type
    void *kf;    // [chunk][key head][4 tiles][DK/32 steps]: K in the call's type
    void *qf;    // the same of Q
    bhalf_t *tm; // [chunk][value head][4 tiles][2 steps][3 parts]: T
    void *pm;    // [chunk][value head][4 tiles][2 steps]: P, two bf16 parts for bf16 calls, else f32
    float *rows; // [chunk][value head][4][64]: factors of the rows of K S, of Q S and of U in the state; [3][0] e^c_n
};

// Parts of a value of the call's type, and of P, the state and the corrected values where only the output takes them.
template <typename T>
constexpr int parts_of() { return std::is_same_v<T, bhalf_t> ? 1 : std::is_same_v<T, half_t> ? 2 : 3; }
template <typename T>
constexpr int out_parts() { return std::is_same_v<T, bhalf_t> ? 2 : 3; }

// P as it is kept for a product: bf16 calls split it once, when it is formed.
template <typename T>
struct DeltaP {
    vec<float, 8> x;
    __device__ void load(const void *pm, uint64_t fragment, uint32_t lane) {
        x = ((const vec<float, 8> *)pm)[fragment * 64 + lane];
    }
    static __device__ void store(void *pm, uint64_t fragment, uint32_t lane, const vec<float, 8> &y) {
        ((vec<float, 8> *)pm)[fragment * 64 + lane] = y;
    }
};
template <>
struct DeltaP<bhalf_t> {
    vec<bhalf_t, 8> x[2];
    __device__ void load(const void *pm, uint64_t fragment, uint32_t lane) {
#pragma unroll
        for (int p = 0; p < 2; p++) x[p] = ((const vec<bhalf_t, 8> *)pm)[(fragment * 2 + p) * 64 + lane];
    }
    static __device__ void store(void *pm, uint64_t fragment, uint32_t lane, const vec<float, 8> &y);
};

constexpr int delta_dim(uint32_t key_dim) { return key_dim <= 64 ? 64 : key_dim <= 128 ? 128 : 256; }

constexpr uint32_t FRAGMENT = 512, SQUARE = 4 * 2 * FRAGMENT; // values of a fragment, of a 64 x 64 operand
constexpr uint32_t key_size(uint32_t dk) { return CHUNK * dk; } // of a chunk's K, Q or K^T

// Chunks of sequence s start here: no two sequences share one.
__device__ inline uint32_t first_chunk(const DeltaArgs &a, uint32_t s) { return first_row(a, s) / CHUNK + s; }

typedef vec<bhalf_t, 8> bf16x8;
typedef vec<bhalf_t, 4> bf16x4;

__device__ inline f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// acc += x y for operands in parts, without the products of parts that lie LEVELS or more steps down. Sums of equal size
// go to one accumulator each, so that no chain is longer than it has to be; the caller adds them.
template <int LEVELS = 3, int NX, int NY, int NA>
__device__ inline void mma_parts(const bf16x8 (&x)[NX], const bf16x8 (&y)[NY], f32x4 (&acc)[NA]) {
#pragma unroll
    for (int i = 0; i < NX; i++)
#pragma unroll
        for (int j = 0; j < NY; j++)
            if (i + j < LEVELS) acc[i + j < NA ? i + j : NA - 1] = mma(x[i], y[j], acc[i + j < NA ? i + j : NA - 1]);
}

__device__ inline float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// Eight consecutive values of a row as they are.
template <bool WIDE, typename T>
__device__ inline vec<T, 8> load8(const T *p) {
    vec<T, 8> x;
    if constexpr (WIDE) {
        constexpr int PER = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < 8; i += PER) {
            const vec<T, PER> v = *(const vec<T, PER> *)(p + i);
#pragma unroll
            for (int j = 0; j < PER; j++) x[i + j] = v[j];
        }
    } else
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = p[i];
    return x;
}

template <int NP, typename T>
__device__ inline void split8(const vec<T, 8> &x, bf16x8 (&part)[NP]) {
    if constexpr (std::is_same_v<T, bhalf_t>) part[0] = x;
    else
#pragma unroll
        for (int j = 0; j < 8; j++) {
            float y = (float)x[j];
#pragma unroll
            for (int p = 0; p < NP; p++) {
                part[p][j] = (bhalf_t)y;
                if (p + 1 < NP) y -= (float)part[p][j];
            }
        }
}

__device__ inline void DeltaP<bhalf_t>::store(void *pm, uint64_t fragment, uint32_t lane, const vec<float, 8> &y) {
    bf16x8 part[2];
    split8(y, part);
#pragma unroll
    for (int p = 0; p < 2; p++) ((bf16x8 *)pm)[(fragment * 2 + p) * 64 + lane] = part[p];
}

// Four consecutive f32 values into the rows of their parts, `apart` values from part to part. All parts but the last are
// cut off, not rounded (a bit mask instead of a conversion each way): three hold 24 bits either way, two 16.
template <int NP>
__device__ inline void split_store(bhalf_t *to, uint32_t apart, f32x4 x) {
#pragma unroll
    for (int p = 0; p < NP; p++) {
        if (p + 1 < NP) {
            uint32_t u[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                u[i] = __float_as_uint(x[i]);
                x[i] -= __uint_as_float(u[i] & 0xFFFF0000u);
            }
            *(uint2 *)(to + p * apart) = make_uint2(__builtin_amdgcn_perm(u[1], u[0], 0x07060302u),
                                                    __builtin_amdgcn_perm(u[3], u[2], 0x07060302u));
        } else {
            bf16x4 h;
#pragma unroll
            for (int i = 0; i < 4; i++) h[i] = (bhalf_t)x[i];
            *(bf16x4 *)(to + p * apart) = h;
        }
    }
}

// Values d on of a row of q or k of the chunk; whatever stands there where there is none.
template <bool WIDE, typename T>
__device__ inline vec<T, 8> row_fragment(const T *base, uint64_t stride, uint32_t row, uint32_t rows, uint32_t d, uint32_t dim) {
    return load8<WIDE>(base + (uint64_t)(row < rows ? row : rows - 1) * stride + (d < dim ? d : 0));
}

// Calls f with true or false, known to the compiler: no load stands behind a branch of its own.
template <typename F>
__device__ inline void with_flag(bool x, F f) {
    if (x) f(std::true_type{});
    else f(std::false_type{});
}

// One workgroup a chunk and value head. The two Gram matrices are a row tile a
// wave; the inverse of 1 + L goes by 16 x 16 blocks: the four diagonal ones by
// substitution, a lane a column, the rest column by column of blocks,
// X_ij = -D_i sum_k L_ik X_kj, in f32 products whose results are the next product's
// operand where they stand. Bound by what it writes and its chain of small steps;
// four workgroups share a CU. 8192 bf16 tokens of 16 / 32 heads of 128: 74 us, about
// 290 MB read and written (4.0 TB/s).
template <typename T, int DK>
__global__ void __launch_bounds__(256, DK <= 128 && sizeof(T) == 2 ? 4 : 2) k_delta_prepare(DeltaArgs a, DeltaWork w) {
    constexpr int NP = parts_of<T>(), STEPS = DK / 32, LS = 68, KS = DK + 16 / (int)sizeof(T);
    constexpr size_t K_BYTES = (size_t)CHUNK * KS * sizeof(T), L_BYTES = CHUNK * LS * 4;
    __shared__ __attribute__((aligned(16))) uint8_t lds[2 * L_BYTES > K_BYTES ? 2 * L_BYTES : K_BYTES];
    __shared__ double sums[CHUNK];
    __shared__ float betas[CHUNK], knorm[CHUNK], qnorm[CHUNK], spoilt[CHUNK];
    const uint32_t tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64);
    const uint32_t col = lane % 16, quad = lane / 16;
    const uint32_t chunk = blockIdx.x / a.value_heads, head = blockIdx.x - chunk * a.value_heads;
    const uint32_t share = a.value_heads / a.key_heads, key_head = head / share;
    // The sequence: the last whose chunks start at or before this one.
    uint32_t s = 0;
    for (uint32_t hi = a.seqs; hi - s > 1;) {
        const uint32_t mid = (s + hi) / 2;
        if (first_chunk(a, mid) <= chunk) s = mid;
        else hi = mid;
    }
    const uint32_t begin = first_row(a, s), end = first_row(a, s + 1), skip = (chunk - first_chunk(a, s)) * CHUNK;
    if (end <= begin || skip >= end - begin) return;
    const uint32_t row0 = begin + skip, rows = min(end - row0, CHUNK);
    const uint64_t at = (uint64_t)chunk * a.value_heads + head;

    // The wave's 16 rows of Q and K, all on their way before the first is used.
    vec<T, 8> xk[STEPS], xq[STEPS];
    with_flag(a.wide, [&](auto wide) {
        const T *q = (const T *)a.q + (uint64_t)row0 * a.q_row + key_head * a.q_head;
        const T *k = (const T *)a.k + (uint64_t)row0 * a.k_row + key_head * a.k_head;
#pragma unroll
        for (int st = 0; st < STEPS; st++) {
            const uint32_t row = wave * 16 + col, d = st * 32 + quad * 8;
            xk[st] = row_fragment<decltype(wide)::value>(k, a.k_row, row, rows, d, a.key_dim);
            xq[st] = row_fragment<decltype(wide)::value>(q, a.q_row, row, rows, d, a.key_dim);
        }
    });
    if (wave == 0) {
        // Sums of the decays, in powers of two. Below e^-200 every f32 is 0, and the sums stay finite.
        double c = 0.0;
        float b = 0.0f;
        if (lane < rows) {
            const float g = a.g[(uint64_t)(row0 + lane) * a.g_row + head];
            c = (g < -200.0f ? -200.0 : (double)g) * 1.4426950408889634074;
            b = a.beta[(uint64_t)(row0 + lane) * a.beta_row + head];
        }
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const double y = __shfl_up(c, d);
            if ((int)lane >= d) c += y;
        }
        sums[lane] = c;
        // What is not finite must not meet the zeros above the diagonal: it is left out of T, and its row marked.
        const bool fine = fabsf(b) < INFINITY;
        betas[lane] = fine ? b : 0.0f;
        spoilt[lane] = fine ? 0.0f : NAN;
    }
    if (rows != CHUNK || a.key_dim != DK) {
#pragma unroll
        for (int st = 0; st < STEPS; st++)
            if (wave * 16 + col >= rows || st * 32 + quad * 8 >= a.key_dim) xk[st] = xq[st] = vec<T, 8>{};
    }
    const uint64_t keys = ((uint64_t)chunk * a.key_heads + key_head) * key_size(DK);
    const bool first = head % share == 0; // of the key head's workgroups: writes what all share
    float kn = 0.0f, qn = 0.0f;
#pragma unroll
    for (int st = 0; st < STEPS; st++) {
        *(vec<T, 8> *)((T *)lds + (wave * 16 + col) * KS + st * 32 + quad * 8) = xk[st];
        if (first) {
            const uint64_t f = keys + (wave * STEPS + st) * FRAGMENT + lane * 8;
            *(vec<T, 8> *)((T *)w.kf + f) = xk[st];
            *(vec<T, 8> *)((T *)w.qf + f) = xq[st];
        }
#pragma unroll
        for (int j = 0; j < 8; j++) {
            kn = fmaf((float)xk[st][j], (float)xk[st][j], kn);
            qn = fmaf((float)xq[st][j], (float)xq[st][j], qn);
        }
    }
    kn += __shfl_xor(kn, 16), qn += __shfl_xor(qn, 16);
    kn += __shfl_xor(kn, 32), qn += __shfl_xor(qn, 32);
    if (quad == 0) {
        knorm[wave * 16 + col] = a.eps >= 0.0f ? 1.0f / sqrtf(kn + a.eps) : 1.0f;
        qnorm[wave * 16 + col] = a.scale * (a.eps >= 0.0f ? 1.0f / sqrtf(qn + a.eps) : 1.0f);
    }
    __syncthreads();
    // Gram matrices: these rows by the tiles of K up to their own.
    f32x4 kk[4], qk[4];
#pragma unroll
    for (int t = 0; t < 4; t++) kk[t] = qk[t] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int st = 0; st < STEPS; st++) {
        bf16x8 mine_k[NP], mine_q[NP];
        split8(xk[st], mine_k);
        split8(xq[st], mine_q);
#pragma unroll
        for (int t = 0; t < 4; t++) {
            if (t > (int)wave) continue;
            bf16x8 other[NP];
            split8(*(const vec<T, 8> *)((const T *)lds + (t * 16 + col) * KS + st * 32 + quad * 8), other);
            f32x4(&ka)[1] = *(f32x4(*)[1])&kk[t], (&qa)[1] = *(f32x4(*)[1])&qk[t];
            mma_parts(mine_k, other, ka);
            mma_parts(mine_q, other, qa);
        }
    }
    if (first) // K^T, turned in LDS
        for (uint32_t f = wave; f < DK / 16 * 2; f += 4) {
            vec<T, 8> x;
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = ((const T *)lds)[(f % 2 * 32 + quad * 8 + j) * KS + f / 2 * 16 + col];
            *(vec<T, 8> *)((T *)w.kt + keys + f * FRAGMENT + lane * 8) = x;
        }
#pragma unroll
    for (int t = 0; t < 4; t++) { // L in place of kk, P of qk; rows and columns past the chunk's are zeros of both
        const uint32_t j = t * 16 + col;
        const double cj = sums[j];
        const float nj = knorm[j];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint32_t i = wave * 16 + quad * 4 + e;
            const float f = fast_exp2((float)(sums[i] - cj)) * nj;
            qk[t][e] = j <= i ? qnorm[i] * (qk[t][e] * f) : 0.0f;
            const float l = j < i ? betas[i] * (knorm[i] * (kk[t][e] * f)) : 0.0f;
            const bool fine = fabsf(l) < INFINITY;
            if (!fine) spoilt[i] = NAN;
            kk[t][e] = fine ? l : 0.0f;
        }
    }
    __syncthreads(); // the keys are used
    float *L = (float *)lds, *P = L + CHUNK * LS; // [64][LS] each
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint32_t f = (wave * 16 + quad * 4 + e) * LS + t * 16 + col;
            L[f] = kk[t][e], P[f] = qk[t][e];
        }
    __syncthreads();
    // A fragment's eight values out of P or what follows it there.
    auto eight = [&](int tile, int st) {
        vec<float, 8> y;
        const f32x4 *x = (const f32x4 *)(P + (tile * 16 + col) * LS + st * 32 + quad * 8);
#pragma unroll
        for (int j = 0; j < 8; j++) y[j] = x[j / 4][j % 4];
        return y;
    };
    if (wave == 0) { // the diagonal blocks of (1 + L)^-1 in the place of L's: lane 16 b + j has column j of block b
        float x[16];
        float *Lb = L + quad * 16 * LS + quad * 16;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            f32x4 y = {i == (int)col ? 1.0f : 0.0f, 0.0f, 0.0f, 0.0f}; // four sums: the chain is a quarter as long
#pragma unroll
            for (int m = 0; m < i; m += 4) {
                const f32x4 row = *(const f32x4 *)(Lb + i * LS + m); // zeros from the diagonal on
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (m + e < i) y[e] = fmaf(-row[e], x[m + e], y[e]);
            }
            x[i] = (y[0] + y[1]) + (y[2] + y[3]);
        }
#pragma unroll
        for (int i = 0; i < 16; i++) Lb[i * LS + col] = x[i];
    } else { // meanwhile P goes out
#pragma unroll
        for (int tile = 0; tile < 4; tile++)
#pragma unroll
            for (int st = 0; st < 2; st++) {
                if (st * 32 > tile * 16 || (tile ? tile : 1) != (int)wave) continue; // tiles 0 and 1 are the first wave's
                DeltaP<T>::store(w.pm, at * 8 + tile * 2 + st, lane, eight(tile, st));
            }
        if (wave == 3) {
            const double c = sums[lane], whole = sums[CHUNK - 1];
            float *to = w.rows + at * 4 * CHUNK;
            const bool here = lane < rows;
            to[lane] = here ? fast_exp2((float)c) * knorm[lane] + spoilt[lane] : 0.0f;
            to[CHUNK + lane] = here ? fast_exp2((float)c) * qnorm[lane] : 0.0f;
            to[2 * CHUNK + lane] = here ? fast_exp2((float)(whole - c)) * knorm[lane] : 0.0f;
            if (lane == 0) to[3 * CHUNK] = fast_exp2((float)whole);
        }
    }
    __syncthreads();
    f32x4 X[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        X[i] = f32x4{0, 0, 0, 0};
        if (i < (int)wave) continue;
        if (i == (int)wave) {
#pragma unroll
            for (int e = 0; e < 4; e++) X[i][e] = L[(i * 16 + quad * 4 + e) * LS + i * 16 + col];
            continue;
        }
        f32x4 sum = {0, 0, 0, 0};
#pragma unroll
        for (int m = 0; m < i; m++) {
            if (m < (int)wave) continue;
            const f32x4 x = *(const f32x4 *)(L + (i * 16 + col) * LS + m * 16 + quad * 4);
#pragma unroll
            for (int e = 0; e < 4; e++) sum = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], X[m][e], sum, 0, 0, 0);
        }
        const f32x4 d = *(const f32x4 *)(L + (i * 16 + col) * LS + i * 16 + quad * 4);
#pragma unroll
        for (int e = 0; e < 4; e++) X[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(-d[e], sum[e], X[i], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) // block (i, wave) of the inverse, times beta of its columns
#pragma unroll
        for (int e = 0; e < 4; e++) P[(i * 16 + quad * 4 + e) * LS + wave * 16 + col] = X[i][e] * betas[wave * 16 + col];
    __syncthreads();
#pragma unroll
    for (int st = 0; st < 2; st++) {
        if (st * 32 > (int)wave * 16) continue; // all zeros, not read
        bf16x8 part[3];
        split8(eight(wave, st), part);
#pragma unroll
        for (int p = 0; p < 3; p++)
            *(bf16x8 *)(w.tm + (at * 8 + wave * 2 + st) * 3 * FRAGMENT + p * FRAGMENT + lane * 8) = part[p];
    }
}

// What one chunk's step reads.
template <typename T, int DK>
struct DeltaChunk {
    vec<T, 8> k[DK / 32], kt[DK / 64][2]; // k: Q for the output's waves
    bf16x8 t[2][3];
    DeltaP<T> p[2];
    f32x4 of_k, of_q, of_u;
    float keep;
    uint32_t v[4]; // a value a register
};

// A workgroup has 16 columns of one head's state. Four waves carry the state, wave
// w the rows DK/4 w on, and of a chunk's tokens the 16 w on: K S, the corrected
// values and the new state, which pass between them through LDS as operands in
// parts (three barriers a chunk). Four more waves follow with the output: Q S beside
// U, P U beside the new state, their stores beside the next chunk's K S (P U there
// too took 8192 tokens 317 us instead of 305). Everything else comes from memory,
// loaded while the chunk before is computed. Bound by the first four's chain: LDS, the
// products (36 of 16 cycles) and the barriers: 2.0 us a chunk, 250 us for 8192
// tokens of 32 heads of 128 x 128, where the 256 workgroups have a CU each.
// Registers for two workgroups a CU spill, and gain only where there are more:
// 16 sequences of 64 tokens 82.6 -> 70.9 us with them, one of 8192 305 -> 338 (both
// with P in one part). f32 with more than 128 key dims spills as it is (256 bytes a
// lane): 10 us a chunk.
constexpr uint32_t DELTA_CHUNK_THREADS = 512;
template <typename T, int DK>
__global__ void __launch_bounds__(DELTA_CHUNK_THREADS) k_delta_chunks(DeltaArgs a, DeltaWork w) {
    constexpr int NP = parts_of<T>(), NO = out_parts<T>(), STEPS = DK / 32, TILES = DK / 64, SS = DK + 8, TS = 72;
    __shared__ __attribute__((aligned(16))) bhalf_t state[3][16 * SS], right[3][16 * TS], values[NO][16 * TS], update[3][16 * TS];
    __shared__ uint32_t spoilt[2][16]; // of every other chunk, a column's first token whose right side is not finite
    const uint32_t tid = threadIdx.x, lane = tid % 64, all = __builtin_amdgcn_readfirstlane(tid / 64), wave = all % 4;
    const bool follows = all >= 4; // with the output
    const uint32_t col = lane % 16, quad = lane / 16;
    // The column groups of one head are eight workgroups apart: on one XCD, whose L2 then has what they share.
    const uint32_t slices = a.value_dim / 16, job = blockIdx.x / (8 * slices) * 8 + blockIdx.x % 8;
    const uint32_t slice = blockIdx.x / 8 % slices, s = job / a.value_heads, head = job - s * a.value_heads;
    if (s >= a.seqs) return;
    const uint32_t key_head = head / (a.value_heads / a.key_heads), dv = slice * 16 + col;
    const uint32_t begin = first_row(a, s), end = max(first_row(a, s + 1), begin), chunk0 = first_chunk(a, s);
    const uint32_t n = end - begin, chunks = (n + CHUNK - 1) / CHUNK;
    const int32_t in = a.slots_in[s], to = a.slots_out[s];
    const uint64_t size = (uint64_t)a.key_dim * a.value_dim;

    f32x4 S[TILES]; // rows (wave * TILES + tile) * 16 + 4 quad + i, column dv
    auto publish = [&] {
#pragma unroll
        for (int m = 0; m < TILES; m++) {
            const uint32_t r = (wave * TILES + m) * 16 + quad * 4;
            split_store<3>(state[0] + col * SS + r, 16 * SS, S[m]);
        }
    };
    if (!follows) {
#pragma unroll
        for (int m = 0; m < TILES; m++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t r = (wave * TILES + m) * 16 + quad * 4 + i;
                float x = in >= 0 && r < a.key_dim ? NAN : 0.0f;
                if (in >= 0 && (uint64_t)in < a.state_slots && r < a.key_dim)
                    x = a.states[((uint64_t)in * a.value_heads + head) * size + (uint64_t)r * a.value_dim + dv];
                S[m][i] = x;
            }
        publish();
        if (tid < 16) spoilt[0][tid] = CHUNK;
    }

    // Addresses are the wave's plus the lane's share.
    auto fragment = [&](const auto *p) {
        using V = std::remove_cv_t<std::remove_reference_t<decltype(*p)>>;
        return ((const vec<V, 8> *)p)[lane];
    };
    // A chunk's operands, each loaded as soon as the chunk before has used its registers: a whole step ahead, and spread
    // over the step (a burst of them fills the path to the L1 and holds the wave up). No load is conditional (past the
    // end the last chunk is loaded again), so that a wait is a count that leaves later loads on their way.
    DeltaChunk<T, DK> x;
    auto key_at = [&](uint32_t c) { return ((uint64_t)(chunk0 + c) * a.key_heads + key_head) * key_size(DK); };
    auto head_at = [&](uint32_t c) { return (uint64_t)(chunk0 + c) * a.value_heads + head; };
    auto factors = [&](uint32_t c, uint32_t which) {
        return ((const f32x4 *)(w.rows + head_at(c) * 4 * CHUNK) + which * (CHUNK / 4) + wave * 4)[quad];
    };
    const T *rows_of = (const T *)(follows ? w.qf : w.kf);
    auto load_k = [&](uint32_t c, int st) { x.k[st] = fragment(rows_of + key_at(c) + (wave * STEPS + st) * FRAGMENT); };
    // The lane's four tokens of a chunk: their rows' offsets, past the chunk's end its last row again (T has zeros there).
    const uint32_t token = wave * 16 + quad * 4;
    const T *v = (const T *)a.v + (uint64_t)begin * a.v_row + head * a.v_head + dv;
    uint64_t v_off[4];
#pragma unroll
    for (int i = 0; i < 4; i++) v_off[i] = (uint64_t)(token + i) * a.v_row;
    auto load_v = [&](uint32_t c) {
        const uint32_t rows = min(n - c * CHUNK, CHUNK);
        const T *vc = v + (uint64_t)(c * CHUNK) * a.v_row;
        uint64_t off[4];
#pragma unroll
        for (int i = 0; i < 4; i++) off[i] = v_off[i];
        if (rows != CHUNK) {
#pragma unroll
            for (int i = 0; i < 4; i++) off[i] = (uint64_t)min(token + i, rows - 1) * a.v_row;
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            using U = std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t>;
            x.v[i] = *(const U *)(vc + off[i]);
        }
        x.of_k = factors(c, 0);
    };
    // Waves 0 and 1 have only zeros in the second step of T and P, which are not written: they load the first again and
    // leave it out.
    const uint32_t second = wave < 2 ? 0 : 1;
    auto load_t = [&](uint32_t c, int st) {
#pragma unroll
        for (int p = 0; p < 3; p++)
            x.t[st][p] = fragment(w.tm + (head_at(c) * 8 + wave * 2 + (st ? second : 0)) * 3 * FRAGMENT + p * FRAGMENT);
    };
    auto load_p = [&](uint32_t c, int st) {
        x.p[st].load(w.pm, head_at(c) * 8 + wave * 2 + (st ? second : 0), lane);
    };
    auto load_kt = [&](uint32_t c, int m, int st) {
        x.kt[m][st] = fragment((const T *)w.kt + key_at(c) + ((wave * TILES + m) * 2 + st) * FRAGMENT);
    };
    auto load_keep = [&](uint32_t c) { x.keep = w.rows[head_at(c) * 4 * CHUNK + 3 * CHUNK]; };
    const uint32_t mine = col * TS + token;
    // What waits for a later load stays behind the barrier it is written behind.
    auto barrier = [] {
        __builtin_amdgcn_sched_barrier(0);
        __syncthreads();
        __builtin_amdgcn_sched_barrier(0);
    };

    // (K or Q) S for the wave's 16 tokens, from the first N parts of the state.
    auto times_state = [&](auto parts, uint32_t next, f32x4(&acc)[3]) {
        constexpr int N = decltype(parts)::value;
        bf16x8 b[STEPS][N];
#pragma unroll
        for (int st = 0; st < STEPS; st++)
#pragma unroll
            for (int p = 0; p < N; p++) b[st][p] = *(const bf16x8 *)(state[p] + col * SS + st * 32 + quad * 8);
#pragma unroll
        for (int i = 0; i < 3; i++) acc[i] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int st = 0; st < STEPS; st++) {
            bf16x8 kp[NP];
            split8(x.k[st], kp);
            mma_parts(kp, b[st], acc);
            load_k(next, st);
        }
    };
    // From a token on that holds what is not finite its columns are NaN, and no token before it is touched: it takes part
    // as a zero (T is triangular, so it reaches none before), and the outputs from there on and the state are replaced.
    auto right_side = [&](uint32_t c, uint32_t next) { // R = V - K S
        f32x4 ks[3], r;
        times_state(std::integral_constant<int, 3>{}, next, ks);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            using U = std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t>;
            r[i] = (float)__builtin_bit_cast(T, (U)x.v[i]) - x.of_k[i] * (ks[0][i] + (ks[1][i] + ks[2][i]));
        }
        uint32_t from = CHUNK;
#pragma unroll
        for (int i = 3; i >= 0; i--)
            if (!(fabsf(r[i]) < INFINITY)) from = token + i, r[i] = 0.0f;
        if (from < CHUNK) atomicMin(&spoilt[c % 2][col], from);
        split_store<3>(right[0] + mine, 16 * TS, r);
        load_v(next);
    };
    auto correct = [&](uint32_t c, uint32_t next) { // U = T R
        if (tid < 16) spoilt[(c + 1) % 2][tid] = CHUNK;
        f32x4 u[3];
        u[0] = u[1] = u[2] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int st = 0; st < 2; st++) {
            if (st <= (int)second) {
                bf16x8 b[3];
#pragma unroll
                for (int p = 0; p < 3; p++) b[p] = *(const bf16x8 *)(right[p] + col * TS + st * 32 + quad * 8);
                mma_parts(x.t[st], b, u);
            }
            load_t(next, st);
        }
        u[0] += u[1] + u[2];
        split_store<3>(update[0] + mine, 16 * TS, u[0] * x.of_u);
        split_store<NO>(values[0] + mine, 16 * TS, u[0]);
        x.of_u = factors(next, 2);
    };
    auto renew = [&](uint32_t c, uint32_t next) { // the state
        const bool ends = spoilt[c % 2][col] < CHUNK;
        f32x4 add[TILES][3];
#pragma unroll
        for (int m = 0; m < TILES; m++) {
            add[m][0] = S[m] * x.keep;
            add[m][1] = add[m][2] = f32x4{0, 0, 0, 0};
        }
        load_keep(next);
#pragma unroll
        for (int st = 0; st < 2; st++) {
            bf16x8 b[3];
#pragma unroll
            for (int p = 0; p < 3; p++) b[p] = *(const bf16x8 *)(update[p] + col * TS + st * 32 + quad * 8);
#pragma unroll
            for (int m = 0; m < TILES; m++) {
                bf16x8 kp[NP];
                split8(x.kt[m][st], kp);
                mma_parts(kp, b, add[m]);
                load_kt(next, m, st);
            }
        }
#pragma unroll
        for (int m = 0; m < TILES; m++) S[m] = ends ? f32x4{NAN, NAN, NAN, NAN} : add[m][0] + (add[m][1] + add[m][2]);
        publish();
    };
    f32x4 qs[3];
    uint64_t out_off[4];
#pragma unroll
    for (int i = 0; i < 4; i++) out_off[i] = (uint64_t)(token + i) * a.out_row;
    f32x4 o[3];
    auto output = [&](uint32_t c, uint32_t next) { // out = Q S + P U of a chunk whose Q S stands in qs
        o[0] = (qs[0] + (qs[1] + qs[2])) * x.of_q, o[1] = o[2] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int st = 0; st < 2; st++) {
            if (st <= (int)second) {
                bf16x8 b[NO];
#pragma unroll
                for (int i = 0; i < NO; i++) b[i] = *(const bf16x8 *)(values[i] + col * TS + st * 32 + quad * 8);
                if constexpr (std::is_same_v<T, bhalf_t>) mma_parts<2>(x.p[st].x, b, o);
                else {
                    bf16x8 p[3];
                    split8(x.p[st].x, p);
                    mma_parts(p, b, o);
                }
            }
            load_p(next, st);
        }
        x.of_q = factors(next, 1);
    };
    auto write = [&](uint32_t c) { // behind the next barrier, where these waves have nothing else to do
        const uint32_t rows = min(n - c * CHUNK, CHUNK), from = spoilt[c % 2][col];
        T *out = (T *)a.out + (uint64_t)(begin + c * CHUNK) * a.out_row + head * a.out_head + dv;
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (token + i < rows) out[out_off[i]] = (T)(token + i < from ? o[0][i] + (o[1][i] + o[2][i]) : NAN);
    };

    // Each kind of wave has a loop of its own, of the same three barriers a chunk (a barrier counts the workgroup's waves,
    // whichever instruction they wait at): in a common one a wait for one kind's loads would be held to the other's too.
    // First loads go in the order of the steps' own: a wait in the loop has to hold for the first step too.
    if (follows) {
        if (chunks > 0) {
            load_p(0, 0), load_p(0, 1);
            x.of_q = factors(0, 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int st = 0; st < STEPS; st++) load_k(0, st);
        }
        barrier();
        for (uint32_t c = 0; c < chunks; c++) {
            if (c) write(c - 1); // its first bad tokens stand until the next barrier
            barrier();
            times_state(std::integral_constant<int, NO>{}, min(c + 1, chunks - 1), qs); // before this chunk, until the next
            barrier();
            output(c, min(c + 1, chunks - 1));
            barrier();
        }
        if (chunks > 0) write(chunks - 1);
        return;
    }
    if (chunks > 0) {
#pragma unroll
        for (int st = 0; st < STEPS; st++) load_k(0, st);
        __builtin_amdgcn_sched_barrier(0);
        load_v(0);
        __builtin_amdgcn_sched_barrier(0);
        load_t(0, 0), load_t(0, 1);
        x.of_u = factors(0, 2);
        __builtin_amdgcn_sched_barrier(0);
        load_keep(0);
#pragma unroll
        for (int st = 0; st < 2; st++)
#pragma unroll
            for (int m = 0; m < TILES; m++) load_kt(0, m, st);
    }
    barrier();
    for (uint32_t c = 0; c < chunks; c++) {
        const uint32_t next = min(c + 1, chunks - 1);
        right_side(c, next);
        barrier();
        correct(c, next);
        barrier();
        renew(c, next);
        barrier();
    }
    if (to < 0 || (uint64_t)to >= a.state_slots) return;
    float *dst = a.states + ((uint64_t)to * a.value_heads + head) * size + dv;
#pragma unroll
    for (int m = 0; m < TILES; m++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t r = (wave * TILES + m) * 16 + quad * 4 + i;
            if (r < a.key_dim) dst[(uint64_t)r * a.value_dim] = S[m][i];
        }
}

}  // namespace rl
