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
// it is as near as f32 arithmetic. Rounded to fewer bits, where the output is
// bf16: P to one part, the state and the corrected values to two in the products
// that only the output takes. Decays are differences of f64 sums, so that a token
// after a strong decay is as exact as one before.
#pragma once
#include "delta.h"

namespace rl {

constexpr uint32_t CHUNK = 64;

// Operands of the chunks, as fragments: for each of 64 lanes eight values, row
// lane % 16 of a 16-row tile, columns 8 (lane / 16) on of a step of 32.
struct DeltaWork {
    void *kt;    // [chunk][key head][DK/16 tiles][2 steps]: K^T in the call's type
    float *tm;   // [chunk][value head][4 tiles][2 steps]: T
    void *pm;    // [chunk][value head][4 tiles][2 steps]: P, bf16 for bf16 calls, else f32
    float *rows; // [chunk][value head][4][64]: factors of the rows of K S, of Q S and of U in the state; [3][0] e^c_n
};

// Parts of a value of the call's type, of P, and of the state and corrected values where only the output takes them.
template <typename T>
constexpr int parts_of() { return std::is_same_v<T, bhalf_t> ? 1 : std::is_same_v<T, half_t> ? 2 : 3; }
template <typename T>
constexpr int out_parts() { return std::is_same_v<T, bhalf_t> ? 2 : 3; }
template <typename T>
using p_type = std::conditional_t<std::is_same_v<T, bhalf_t>, bhalf_t, float>;

constexpr int delta_dim(uint32_t key_dim) { return key_dim <= 64 ? 64 : key_dim <= 128 ? 128 : 256; }

constexpr uint32_t FRAGMENT = 512, SQUARE = 4 * 2 * FRAGMENT; // values of a fragment, of a 64 x 64 operand
constexpr uint32_t kt_size(uint32_t dk) { return dk / 16 * 2 * FRAGMENT; }

// Chunks of sequence s start here: no two sequences share one.
__device__ inline uint32_t first_chunk(const DeltaArgs &a, uint32_t s) { return first_row(a, s) / CHUNK + s; }

typedef vec<bhalf_t, 8> bf16x8;
typedef vec<bhalf_t, 4> bf16x4;

__device__ inline f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// acc += x y for operands in parts, without the products of parts that lie three or more steps down. Sums of equal size
// go to one accumulator each, so that no chain is longer than it has to be; the caller adds them.
template <int NX, int NY, int NA>
__device__ inline void mma_parts(const bf16x8 (&x)[NX], const bf16x8 (&y)[NY], f32x4 (&acc)[NA]) {
#pragma unroll
    for (int i = 0; i < NX; i++)
#pragma unroll
        for (int j = 0; j < NY; j++)
            if (i + j < 3) acc[i + j < NA ? i + j : NA - 1] = mma(x[i], y[j], acc[i + j < NA ? i + j : NA - 1]);
}

__device__ inline float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// Eight consecutive values of a row as they are.
template <typename T>
__device__ inline vec<T, 8> load8(const T *p, bool wide) {
    vec<T, 8> x;
    if (wide) {
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

// Four consecutive f32 values into the rows of their parts, `apart` values from part to part.
template <int NP>
__device__ inline void split_store(bhalf_t *to, uint32_t apart, f32x4 x) {
#pragma unroll
    for (int p = 0; p < NP; p++) {
        bf16x4 h;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            h[i] = (bhalf_t)x[i];
            x[i] -= (float)h[i];
        }
        *(bf16x4 *)(to + p * apart) = h;
    }
}

// Values 8 (lane / 16) on of a step of q or k, of a row of the chunk; whatever stands there where there is none.
template <typename T>
__device__ inline vec<T, 8> row_fragment(const T *base, uint64_t stride, uint32_t row, uint32_t rows, uint32_t d, uint32_t dim,
                                         bool wide) {
    return load8(base + (uint64_t)(row < rows ? row : rows - 1) * stride + (d < dim ? d : 0), wide);
}

// One workgroup a chunk and value head. The two Gram matrices are a row tile a
// wave; the inverse of 1 + L goes by 16 x 16 blocks: the four diagonal ones by
// substitution, a lane a column, the rest column by column of blocks,
// X_ij = -D_i sum_k L_ik X_kj, in f32 products whose results are the next product's
// operand where they stand. Bound by its chain of small steps; four workgroups
// share a CU.
template <typename T, int DK>
__global__ void __launch_bounds__(256, DK <= 128 && sizeof(T) == 2 ? 4 : 2) k_delta_prepare(DeltaArgs a, DeltaWork w) {
    using TP = p_type<T>;
    constexpr int NP = parts_of<T>(), STEPS = DK / 32, LS = 68, KS = DK + 16 / (int)sizeof(T);
    constexpr size_t K_BYTES = (size_t)CHUNK * KS * sizeof(T), L_BYTES = CHUNK * LS * 4, D_BYTES = 4 * 16 * 20 * 4;
    __shared__ __attribute__((aligned(16))) uint8_t lds[L_BYTES + D_BYTES > K_BYTES ? L_BYTES + D_BYTES : K_BYTES];
    __shared__ double sums[CHUNK];
    __shared__ float betas[CHUNK], knorm[CHUNK], qnorm[CHUNK];
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
    const bool clean = rows == CHUNK && a.key_dim == DK;
    const T *q = (const T *)a.q + (uint64_t)row0 * a.q_row + key_head * a.q_head;
    const T *k = (const T *)a.k + (uint64_t)row0 * a.k_row + key_head * a.k_head;
    const uint64_t at = (uint64_t)chunk * a.value_heads + head;

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
        betas[lane] = b;
    }
    // Gram matrices, the wave's 16 rows by the tiles up to its own.
    auto fragment = [&](const T *base, uint64_t stride, int tile, int st) {
        const uint32_t row = tile * 16 + col, d = st * 32 + quad * 8;
        vec<T, 8> x = row_fragment(base, stride, row, rows, d, a.key_dim, a.wide);
        if (!clean && (row >= rows || d >= a.key_dim)) x = vec<T, 8>{};
        return x;
    };
    f32x4 kk[4], qk[4];
#pragma unroll
    for (int t = 0; t < 4; t++) kk[t] = qk[t] = f32x4{0, 0, 0, 0};
    float kn = 0.0f, qn = 0.0f;
#pragma unroll
    for (int st = 0; st < STEPS; st++) {
        const vec<T, 8> xk = fragment(k, a.k_row, wave, st), xq = fragment(q, a.q_row, wave, st);
        *(vec<T, 8> *)((T *)lds + (wave * 16 + col) * KS + st * 32 + quad * 8) = xk;
        bf16x8 mine_k[NP], mine_q[NP];
        split8(xk, mine_k);
        split8(xq, mine_q);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            kn = fmaf((float)xk[j], (float)xk[j], kn);
            qn = fmaf((float)xq[j], (float)xq[j], qn);
        }
#pragma unroll
        for (int t = 0; t < 4; t++) {
            if (t > (int)wave) continue;
            bf16x8 other[NP];
            split8(fragment(k, a.k_row, t, st), other);
            f32x4(&ka)[1] = *(f32x4(*)[1])&kk[t], (&qa)[1] = *(f32x4(*)[1])&qk[t];
            mma_parts(mine_k, other, ka);
            mma_parts(mine_q, other, qa);
        }
    }
    kn += __shfl_xor(kn, 16), qn += __shfl_xor(qn, 16);
    kn += __shfl_xor(kn, 32), qn += __shfl_xor(qn, 32);
    if (quad == 0) {
        knorm[wave * 16 + col] = a.eps >= 0.0f ? 1.0f / sqrtf(kn + a.eps) : 1.0f;
        qnorm[wave * 16 + col] = a.scale * (a.eps >= 0.0f ? 1.0f / sqrtf(qn + a.eps) : 1.0f);
    }
    __syncthreads();
    // K^T, turned in LDS, by the first of the key head's workgroups.
    if (head % share == 0) {
        T *kt = (T *)w.kt + ((uint64_t)chunk * a.key_heads + key_head) * kt_size(DK);
        for (uint32_t f = wave; f < DK / 16 * 2; f += 4) {
            vec<T, 8> x;
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = ((const T *)lds)[(f % 2 * 32 + quad * 8 + j) * KS + f / 2 * 16 + col];
            *(vec<T, 8> *)(kt + f * FRAGMENT + lane * 8) = x;
        }
    }
    if (wave == 1) {
        const double c = sums[lane], whole = sums[CHUNK - 1];
        float *to = w.rows + at * 4 * CHUNK;
        const bool here = lane < rows;
        to[lane] = here ? fast_exp2((float)c) * knorm[lane] : 0.0f;
        to[CHUNK + lane] = here ? fast_exp2((float)c) * qnorm[lane] : 0.0f;
        to[2 * CHUNK + lane] = here ? fast_exp2((float)(whole - c)) * knorm[lane] : 0.0f;
        if (lane == 0) to[3 * CHUNK] = fast_exp2((float)whole);
    }
    __syncthreads();
    // P goes out through LDS, then L takes its place.
    float *L = (float *)lds, *D = (float *)(lds + L_BYTES); // [64][LS]; [4][16][20]
    f32x4 l[4];
#pragma unroll
    for (int t = 0; t < 4; t++) {
        const uint32_t j = t * 16 + col;
        const double cj = sums[j];
        const float nj = knorm[j];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint32_t i = wave * 16 + quad * 4 + e;
            float p = 0.0f;
            l[t][e] = 0.0f;
            if (j <= i) { // rows and columns past the chunk's are zeros of kk and qk
                const float f = fast_exp2((float)(sums[i] - cj)) * nj;
                p = qnorm[i] * (qk[t][e] * f);
                if (j < i) l[t][e] = betas[i] * (knorm[i] * (kk[t][e] * f));
            }
            L[i * LS + j] = p;
        }
    }
    __syncthreads();
    auto write_out = [&](auto *to) { // a wave a row tile, from its own rows of LDS
        using V = std::remove_reference_t<decltype(*to)>;
#pragma unroll
        for (uint32_t st = 0; st < 2; st++) {
            if (st * 32 > wave * 16) continue; // all zeros, not read
            const float *x = L + (wave * 16 + col) * LS + st * 32 + quad * 8;
            vec<V, 8> y;
#pragma unroll
            for (int j = 0; j < 8; j++) y[j] = (V)x[j];
            *(vec<V, 8> *)(to + (wave * 2 + st) * FRAGMENT + lane * 8) = y;
        }
    };
    write_out((TP *)w.pm + at * SQUARE);
    __syncthreads();
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) L[(wave * 16 + quad * 4 + e) * LS + t * 16 + col] = l[t][e];
    __syncthreads();
    if (wave == 0) { // D = (1 + L)^-1 of the diagonal blocks: lane 16 b + j has column j of block b
        float x[16];
        const float *Lb = L + quad * 16 * LS + quad * 16;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            float y = i == (int)col ? 1.0f : 0.0f;
#pragma unroll
            for (int m = 0; m < i; m += 4) {
                const f32x4 row = *(const f32x4 *)(Lb + i * LS + m); // zeros from the diagonal on
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (m + e < i) y = fmaf(-row[e], x[m + e], y);
            }
            x[i] = y;
        }
#pragma unroll
        for (int i = 0; i < 16; i++) D[(quad * 16 + i) * 20 + col] = x[i];
    }
    __syncthreads();
    f32x4 X[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        X[i] = f32x4{0, 0, 0, 0};
        if (i < (int)wave) continue;
        if (i == (int)wave) {
#pragma unroll
            for (int e = 0; e < 4; e++) X[i][e] = D[(i * 16 + quad * 4 + e) * 20 + col];
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
        const f32x4 d = *(const f32x4 *)(D + (i * 16 + col) * 20 + quad * 4);
#pragma unroll
        for (int e = 0; e < 4; e++) X[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(-d[e], sum[e], X[i], 0, 0, 0);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; i++) // block (i, wave) of the inverse, times beta of its columns
#pragma unroll
        for (int e = 0; e < 4; e++) L[(i * 16 + quad * 4 + e) * LS + wave * 16 + col] = X[i][e] * betas[wave * 16 + col];
    __syncthreads();
    write_out(w.tm + at * SQUARE);
}

// What one chunk's step reads.
template <typename T, int DK>
struct DeltaChunk {
    vec<T, 8> k[DK / 32], q[DK / 32], kt[DK / 64][2];
    vec<float, 8> t[2];
    vec<p_type<T>, 8> p[2];
    f32x4 of_k, of_q, of_u;
    float keep;
    T v[4];
};

// A workgroup has 16 columns of one head's state, wave w the rows DK/4 w on, and
// of a chunk's tokens the 16 w on. State, right-hand sides and corrected values
// pass between the waves through LDS as operands in parts (three barriers a chunk);
// everything else comes from memory, loaded while the chunk two before is computed.
// Bound by the chain of a chunk: the products of a wave, and the three exchanges.
template <typename T, int DK>
__global__ void __launch_bounds__(256) k_delta_chunks(DeltaArgs a, DeltaWork w) {
    constexpr int NP = parts_of<T>(), NO = out_parts<T>(), STEPS = DK / 32, TILES = DK / 64, SS = DK + 8, TS = 72;
    constexpr bool AHEAD = DK * sizeof(T) <= 512; // two chunks' operands fit the registers
    __shared__ __attribute__((aligned(16))) bhalf_t state[3][16 * SS], right[3][16 * TS], values[NO][16 * TS], update[3][16 * TS];
    const uint32_t tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64);
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
    auto publish = [&] {
#pragma unroll
        for (int m = 0; m < TILES; m++) {
            const uint32_t r = (wave * TILES + m) * 16 + quad * 4;
            split_store<3>(state[0] + col * SS + r, 16 * SS, S[m]);
        }
    };

    const T *q = (const T *)a.q + key_head * a.q_head, *k = (const T *)a.k + key_head * a.k_head;
    const T *v = (const T *)a.v + head * a.v_head + dv;
    auto load = [&](uint32_t c, DeltaChunk<T, DK> &x) {
        const uint64_t row0 = begin + c * CHUNK;
        const uint32_t rows = min(n - c * CHUNK, CHUNK);
#pragma unroll
        for (int st = 0; st < STEPS; st++) {
            const uint32_t d = st * 32 + quad * 8;
            x.k[st] = row_fragment(k + row0 * a.k_row, a.k_row, wave * 16 + col, rows, d, a.key_dim, a.wide);
            x.q[st] = row_fragment(q + row0 * a.q_row, a.q_row, wave * 16 + col, rows, d, a.key_dim, a.wide);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) x.v[i] = v[(row0 + min(wave * 16 + quad * 4 + i, rows - 1)) * a.v_row];
        const uint64_t at = (uint64_t)(chunk0 + c) * a.value_heads + head;
        const float *f = w.rows + at * 4 * CHUNK + wave * 16 + quad * 4;
        x.of_k = *(const f32x4 *)f, x.of_q = *(const f32x4 *)(f + CHUNK), x.of_u = *(const f32x4 *)(f + 2 * CHUNK);
        x.keep = w.rows[at * 4 * CHUNK + 3 * CHUNK];
#pragma unroll
        for (int st = 0; st < 2; st++) {
            if (st * 32 > (int)wave * 16) continue; // all zeros: not written, not used
            const uint64_t f = at * SQUARE + (wave * 2 + st) * FRAGMENT + lane * 8;
            x.t[st] = *(const vec<float, 8> *)(w.tm + f);
            x.p[st] = *(const vec<p_type<T>, 8> *)((const p_type<T> *)w.pm + f);
        }
        const T *kt = (const T *)w.kt + ((uint64_t)(chunk0 + c) * a.key_heads + key_head) * kt_size(DK);
#pragma unroll
        for (int m = 0; m < TILES; m++)
#pragma unroll
            for (int st = 0; st < 2; st++)
                x.kt[m][st] = *(const vec<T, 8> *)(kt + ((wave * TILES + m) * 2 + st) * FRAGMENT + lane * 8);
    };

    auto step = [&](uint32_t c, DeltaChunk<T, DK> &x) {
        const uint32_t rows = min(n - c * CHUNK, CHUNK);
        const bool clean = rows == CHUNK && a.key_dim == DK;
        if (!clean) { // what stands outside the chunk or the head may be anything
#pragma unroll
            for (int st = 0; st < STEPS; st++)
                if (wave * 16 + col >= rows || st * 32 + quad * 8 >= a.key_dim) x.k[st] = x.q[st] = vec<T, 8>{};
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (wave * 16 + quad * 4 + i >= rows) x.v[i] = (T)0.0f;
        }
        // K S and Q S for the wave's tokens.
        f32x4 ks[3], qs[3];
#pragma unroll
        for (int i = 0; i < 3; i++) ks[i] = qs[i] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int st = 0; st < STEPS; st++) {
            bf16x8 b[3], kp[NP], qp[NP];
#pragma unroll
            for (int p = 0; p < 3; p++) b[p] = *(const bf16x8 *)(state[p] + col * SS + st * 32 + quad * 8);
            split8(x.k[st], kp);
            split8(x.q[st], qp);
            mma_parts(kp, b, ks);
            if constexpr (NO == 3) mma_parts(qp, b, qs);
            else {
                bf16x8(&two)[2] = *(bf16x8(*)[2])b;
                mma_parts(qp, two, qs);
            }
        }
        f32x4 r;
#pragma unroll
        for (int i = 0; i < 4; i++) r[i] = (float)x.v[i] - x.of_k[i] * (ks[0][i] + (ks[1][i] + ks[2][i]));
        const uint32_t mine = col * TS + wave * 16 + quad * 4;
        split_store<3>(right[0] + mine, 16 * TS, r);
        bf16x8 t[2][3];
#pragma unroll
        for (int st = 0; st < 2; st++)
            if (st * 32 <= (int)wave * 16) split8(x.t[st], t[st]);
        __syncthreads();
        // U = T R.
        f32x4 u[3];
        u[0] = u[1] = u[2] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int st = 0; st < 2; st++) {
            if (st * 32 > (int)wave * 16) continue;
            bf16x8 b[3];
#pragma unroll
            for (int p = 0; p < 3; p++) b[p] = *(const bf16x8 *)(right[p] + col * TS + st * 32 + quad * 8);
            mma_parts(t[st], b, u);
        }
        u[0] += u[1] + u[2];
        split_store<3>(update[0] + mine, 16 * TS, u[0] * x.of_u);
        split_store<NO>(values[0] + mine, 16 * TS, u[0]);
        __syncthreads();
        // The state, and out = Q S + P U.
        f32x4 add[TILES][3];
#pragma unroll
        for (int m = 0; m < TILES; m++) {
            add[m][0] = S[m] * x.keep;
            add[m][1] = add[m][2] = f32x4{0, 0, 0, 0};
        }
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
            }
        }
#pragma unroll
        for (int m = 0; m < TILES; m++) S[m] = add[m][0] + (add[m][1] + add[m][2]);
        publish();
        f32x4 o[3];
        o[0] = (qs[0] + (qs[1] + qs[2])) * x.of_q, o[1] = o[2] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int st = 0; st < 2; st++) {
            if (st * 32 > (int)wave * 16) continue;
            constexpr int PP = std::is_same_v<T, bhalf_t> ? 1 : 3;
            bf16x8 b[NO], p[PP];
#pragma unroll
            for (int i = 0; i < NO; i++) b[i] = *(const bf16x8 *)(values[i] + col * TS + st * 32 + quad * 8);
            split8(x.p[st], p);
            mma_parts(p, b, o);
        }
        T *out = (T *)a.out + head * a.out_head + dv;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t row = c * CHUNK + wave * 16 + quad * 4 + i;
            if (row < n) out[(uint64_t)(begin + row) * a.out_row] = (T)(o[0][i] + (o[1][i] + o[2][i]));
        }
        __syncthreads();
    };

    publish();
    DeltaChunk<T, DK> x;
    if (chunks > 0) load(0, x);
    if constexpr (AHEAD) {
        DeltaChunk<T, DK> y;
        if (chunks > 1) load(1, y);
        __syncthreads();
        for (uint32_t c = 0; c < chunks; c += 2) {
            step(c, x);
            if (c + 2 < chunks) load(c + 2, x);
            if (c + 1 >= chunks) break;
            step(c + 1, y);
            if (c + 3 < chunks) load(c + 3, y);
        }
    } else {
        __syncthreads();
        for (uint32_t c = 0; c < chunks; c++) {
            step(c, x);
            if (c + 1 < chunks) load(c + 1, x);
        }
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
