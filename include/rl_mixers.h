/*
 * rl_mixers.h — C ABI of the MI355X (gfx950) token mixers: what the layers
 * between the embedding lookup and the output head (rl_head.h) do across the
 * tokens of a sequence. Rotary positions, a paged key-value cache that is
 * quantised as it is written, attention of new tokens over that cache, also behind
 * prefixes that sequences share, the gated delta rule, the short causal convolution
 * and the selective state space scan.
 *
 * Conventions as in rl_sampler.h: status codes, rl_sampler_last_error() for the
 * message, stream-ordered calls that return before the kernels finish, one
 * thread and one stream at a time per handle. Every device buffer that a call
 * needs is allocated by the create functions; the others allocate nothing and
 * may be captured into a graph.
 *
 * Tensors are described by rl_heads: [rows][heads][dim] in device memory with
 * strides in elements, the last axis contiguous. Where data and strides are
 * multiples of 16 bytes they are read and written 16 bytes at a time.
 */
#ifndef RL_MIXERS_H
#define RL_MIXERS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types. RL_I8 and RL_F8 (e4m3 without infinities: 448 is the largest)
 * are cache formats only, with an f32 step per token and head. */
enum { RL_F32 = 0, RL_F16 = 1, RL_BF16 = 2, RL_I8 = 3, RL_F8 = 4 };

typedef struct rl_heads {
    void *data;
    uint64_t row_stride;  /* elements from a row to the next */
    uint64_t head_stride; /* elements from a head to the next */
    uint32_t heads;
    uint32_t dim;
    uint32_t dtype; /* RL_F32, RL_F16 or RL_BF16 */
    uint32_t reserved;
} rl_heads;

/* ------------------------------------------------------------- rotary --
 * The first `dims` values of a head, taken in pairs (a, b), are turned by
 * position * f_i radians for pair i and scaled by the magnitude m:
 *   a' = m (a cos - b sin),  b' = m (a sin + b cos)
 * with f_i = base^(-2 i / dims). Angles are reduced in f64, so they are as exact
 * at position 10^6 as at 1; the products are f32, rounded once to the output's
 * type. Values past `dims` are copied. */
enum { RL_ROTARY_HALF = 0 /* pairs (i, i + dims/2) */, RL_ROTARY_INTERLEAVED = 1 /* pairs (2i, 2i + 1) */ };

/* RL_ROTARY_LINEAR divides every f_i by `factor`; RL_ROTARY_NTK takes
 * base * factor^(dims / (dims - 2)) for the base; RL_ROTARY_YARN divides those of
 * the pairs that turn less than beta_slow times in `original` positions, keeps
 * those that turn more than beta_fast times, and goes from one to the other
 * linearly in the pair's index; its magnitude is 0.1 ln(factor) + 1. */
enum { RL_ROTARY_PLAIN = 0, RL_ROTARY_LINEAR = 1, RL_ROTARY_NTK = 2, RL_ROTARY_YARN = 3 };

typedef struct rl_rotary_spec {
    uint32_t dims;   /* values turned, even, 2 to 512 */
    uint32_t layout;
    uint32_t scaling;
    uint32_t original; /* RL_ROTARY_YARN: the context that the model was trained on */
    double base;       /* above 1 */
    double factor;     /* at least 1; unused by RL_ROTARY_PLAIN */
    double beta_fast, beta_slow; /* RL_ROTARY_YARN; 0 takes 32 and 1 */
    double magnitude;            /* 0 takes the scaling's own */
} rl_rotary_spec;

typedef struct rl_rotary rl_rotary;

int rl_rotary_create(int device, const rl_rotary_spec *spec, rl_rotary **out);
void rl_rotary_destroy(rl_rotary *rotary);

/* Radians a position of each of the dims/2 pairs, and the magnitude (either may
 * be NULL). Host only. */
int rl_rotary_frequencies(const rl_rotary *rotary, double *radians, double *magnitude);

/* Turns `tensors` (1 or 2: queries and keys) inputs of `rows` rows into their
 * outputs in one launch; positions [rows] i64 on the device, any value whose
 * magnitude is below 2^53. out[i] may be in[i] itself (same data, strides and
 * type) or must not overlap it; its type may differ. inverse != 0 turns by the
 * negative angles, which is the gradient with respect to the input of a turn
 * whose output has this gradient, and takes a turn back if the magnitude is 1. */
int rl_rotary_rows(rl_rotary *rotary, const int64_t *positions, uint32_t rows, const rl_heads *in,
                   const rl_heads *out, uint32_t tensors, int inverse, void *stream);

/* -------------------------------------------------------------- cache --
 * Keys and values of `pages` pages of `page` tokens each, for one layer. A
 * token's slot is its page's number times `page` plus its place in the page.
 * Formats: RL_F16 and RL_BF16 hold values rounded once. RL_I8 holds
 * c = rint(x / s) with s = max|x| / 127 over the token's head, RL_F8 holds
 * c = e4m3(x / s) with s = max|x| / 448 (f32, IEEE division, ties to even); a
 * value reads as c * s. A head that holds a NaN or an infinity reads as NaN
 * throughout in these two. */
typedef struct rl_kv_cache rl_kv_cache;

/* dim: 16 to 256, a multiple of 16. page and pages: any from 1; pages * page at
 * most 2^32 tokens, kv_heads at most 2^16. The contents start as zeros. */
int rl_kv_cache_create(int device, uint32_t pages, uint32_t page, uint32_t kv_heads, uint32_t dim, uint32_t format,
                       rl_kv_cache **out);
void rl_kv_cache_destroy(rl_kv_cache *cache);

/* Bytes of device memory the handle holds. */
uint64_t rl_kv_cache_bytes(const rl_kv_cache *cache);

/* Writes rows keys[i], values[i] to slots[i] (i64 [rows] on the device). A slot
 * that is negative or past the cache is left out, so a batch may hold padding. The
 * others are to be distinct: rows are written side by side, so a slot that a call
 * gives twice holds a mixture of the rows' keys, values, codes and steps until it is
 * written again (no other slot is touched by it). With `rotary` the keys are turned
 * by positions[i] first (in f32, before the one rounding); NULL stores them as
 * they are and reads no positions. keys and values have one type and shape. */
int rl_kv_cache_write(rl_kv_cache *cache, const rl_heads *keys, const rl_heads *values, const int64_t *slots,
                      uint32_t rows, const rl_rotary *rotary, const int64_t *positions, void *stream);

/* keys[i], values[i] = what the cache holds at slots[i]. A slot outside the cache
 * gives a row of NaN, as an unknown token does in rl_head_embed_rows. */
int rl_kv_cache_read(rl_kv_cache *cache, const int64_t *slots, uint32_t rows, const rl_heads *keys,
                     const rl_heads *values, void *stream);

/* ---------------------------------------------------------- attention --
 * Sequence s has the query rows starts[s] .. starts[s+1] (its newest tokens,
 * whose keys and values are in the cache already) and lens[s] tokens in the
 * cache, the t-th of them in slot pages[s * table_width + t / page] * page
 * + t % page. Row i of its n rows stands at position lens[s] - n + i and sees the
 * tokens up to its own, with window > 0 the last `window` of them:
 *   out = sum_t softmax_t(scale q . k_t) v_t,  lse = ln sum_t exp(scale q . k_t)
 * Query head h reads the key-value head h / (q_heads / kv_heads). A row that sees
 * nothing gives zeros and an lse of -inf. Scores, softmax and sums are f32; the
 * weights go into the product with the values as sums of 16-bit parts, good to 16
 * bits or more for 16-bit queries and to 22 or more for f32 ones (over f16 values no
 * finer than 2^-33 of the largest weight so far). What a row does not see does not
 * reach it, whatever it holds. An infinity among the f16 or bf16 values that a row
 * sees may read as NaN (a part of its weight may be 0), and so may one among such
 * keys to f32 queries. */
typedef struct rl_attention rl_attention;

/* Workspace for calls of up to max_rows query rows over caches of kv_heads heads
 * and up to max_len tokens a sequence: 8 bytes a row and head, and 4 D + 8 bytes for
 * each partial result (D: dim rounded up to 64, 128 or 256), of which there are about
 * max_rows * q_heads * min(max_len / 1536 + 1, 256), at most 2^20, at least 2^15.
 * q_heads: a multiple of kv_heads; max_rows * q_heads at most 2^23. */
int rl_attention_create(int device, uint32_t max_rows, uint32_t q_heads, uint32_t kv_heads, uint32_t dim,
                        uint32_t max_len, rl_attention **out);
void rl_attention_destroy(rl_attention *attention);

/* q and out: [rows][q_heads][dim] of one type; a cache in RL_F16 takes f16 or f32
 * queries, one in RL_BF16 bf16 or f32, the 8-bit ones all three. starts i32
 * [seqs + 1] rising from 0 to rows, or NULL for one row a sequence (rows == seqs);
 * lens i32 [seqs], a negative one as 0; pages i32 [seqs][table_width]; lse f32
 * [rows][q_heads] or NULL. most_rows and max_len bound the rows and tokens of any one
 * sequence (0: as many as the call has rows, and the handle's max_len); a sequence
 * past either bound, or one that needs a page outside its table or the cache, gives
 * NaN. Only entries of `pages` that hold tokens in sight are read. */
int rl_attention_rows(rl_attention *attention, const rl_kv_cache *cache, const rl_heads *q, const rl_heads *out,
                      float *lse, uint32_t rows, const int32_t *starts, const int32_t *lens, uint32_t seqs,
                      const int32_t *pages, uint32_t table_width, float scale, uint32_t window, uint32_t most_rows,
                      uint32_t max_len, void *stream);

/* The same where sequences share long beginnings, whose keys and values are then read
 * once for a group and not once for each sequence. The sequences group_starts[g] ..
 * group_starts[g + 1] (i32 [groups + 1], rising; what lies before the first or from the
 * last on has no prefix) have the same prefix_lens[g] tokens (i32, a negative one as 0)
 * before their own, the t-th of them in slot
 * prefix_pages[g * prefix_width + t / page] * page + t % page. lens and pages are
 * those of their own tokens, which begin a page: every row sees its whole prefix and its
 * own sequence's tokens up to its own, as above without a window. max_prefix bounds the
 * tokens of any one prefix (0: the handle's max_len); past it the rows of the group are
 * NaN. Rows from starts[seqs] on are not written. rows * q_heads at most 2^20. */
int rl_attention_shared(rl_attention *attention, const rl_kv_cache *cache, const rl_heads *q, const rl_heads *out,
                        float *lse, uint32_t rows, const int32_t *starts, const int32_t *lens, uint32_t seqs,
                        const int32_t *pages, uint32_t table_width, const int32_t *group_starts,
                        const int32_t *prefix_lens, uint32_t groups, const int32_t *prefix_pages, uint32_t prefix_width,
                        float scale, uint32_t most_rows, uint32_t max_len, uint32_t max_prefix, void *stream);

/* --------------------------------------------------------- delta rule --
 * Every value head of a sequence has a state S [key_dim][value_dim], and each
 * token, in order, does
 *   S <- e^g S;  u = beta (v - S^T k);  S <- S + k u^T;  out = scale S^T q
 * with q and k of the key head h / (value_heads / key_heads). norm_eps >= 0
 * divides q and k by sqrt(|x|^2 + norm_eps) first; negative leaves them. State and
 * sums are f32. */
typedef struct rl_delta rl_delta;

/* Workspace for calls of up to max_rows tokens in up to max_seqs sequences: none below
 * 13 rows, else for max_rows / 64 + min(max_seqs, max_rows / 16 + 1) chunks, each of
 * 41 KiB a value head and 768 D bytes a key head (D: key_dim rounded up to 64, 128 or
 * 256). A call of more sequences than its chunks have room for, or of 2^27 columns of
 * states (seqs * value_heads * value_dim) or more, goes token by token.
 * value_heads: a multiple of key_heads. key_dim, value_dim: 16 to 256, multiples of
 * 16. */
int rl_delta_create(int device, uint32_t max_rows, uint32_t max_seqs, uint32_t key_heads, uint32_t value_heads,
                    uint32_t key_dim, uint32_t value_dim, rl_delta **out);
void rl_delta_destroy(rl_delta *delta);

/* q, k [rows][key_heads][key_dim], v, out [rows][value_heads][value_dim] of one
 * type; g (log decay, at most 0 in use) and beta f32 [rows][value_heads] with row
 * strides of their own; starts i32 [seqs + 1] rising from 0 to rows, or NULL for
 * one row a sequence. states f32 [state_slots][value_heads][key_dim][value_dim]:
 * sequence s begins from states[slots_in[s]] (zeros if that is negative) and
 * leaves its state in states[slots_out[s]] (nowhere if that is negative). The two
 * may be equal; else no slot that a sequence of the call reads may be one that
 * another writes, and no two sequences write one slot. A slot from state_slots on reads as NaN and is not written. A
 * sequence without rows passes its state on. most_rows bounds the rows of any one
 * sequence (0: as many as the call has); it may be any number, since it only picks
 * the form that is used for all of them, one token after the other or chunks on the
 * matrix cores. Both are as exact as f32 sums, but do not give the same bits, and in
 * chunks an infinity reads as NaN. What is not finite reaches the tokens after it,
 * none before. */
int rl_delta_rows(rl_delta *delta, const rl_heads *q, const rl_heads *k, const rl_heads *v, const rl_heads *out,
                  const float *g, uint64_t g_stride, const float *beta, uint64_t beta_stride, float *states,
                  uint64_t state_slots, const int32_t *slots_in, const int32_t *slots_out, const int32_t *starts,
                  uint32_t rows, uint32_t seqs, float scale, float norm_eps, uint32_t most_rows, void *stream);

/* -------------------------------------------------- short convolution --
 * Every channel's row is the sum of its last `width` rows:
 *   y[t][c] = act(bias[c] + sum_j weight[c][j] x[t - width + 1 + j][c])
 * with act(y) = y or y / (1 + e^-y). The width - 1 rows before a sequence's first are
 * its state, as they came in. Sums are f32, rounded once to the output's type; below
 * 2^-119 an activated one may be 0. */
enum { RL_CONV_PLAIN = 0, RL_CONV_SILU = 1 };

typedef struct rl_conv rl_conv;

/* weight [channels][width] and bias [channels] (or NULL) f32 on the host, copied. width
 * 2 to 8, channels at most 2^20. */
int rl_conv_create(int device, uint32_t channels, uint32_t width, const float *weight, const float *bias,
                   uint32_t activation, rl_conv **out);
void rl_conv_destroy(rl_conv *conv);

/* x, out [rows][1][channels] of one type; out must not overlap x. starts i32 [seqs + 1]
 * rising from 0 to rows, or NULL for one row a sequence. states [state_slots][width - 1]
 * [channels] of x's type: sequence s has its rows before the first in
 * states[slots_in[s]] (zeros if that is negative) and leaves its last ones, the old ones
 * among them if it is shorter, in states[slots_out[s]] (nowhere if that is negative),
 * under the rules of rl_delta_rows: the two may be equal; else no slot that a sequence
 * reads is one that another writes, and none is written twice. A slot from state_slots
 * on reads as NaN and is not written. A sequence without rows passes its state on, and
 * rows from starts[seqs] on are not written. */
int rl_conv_rows(rl_conv *conv, const rl_heads *x, const rl_heads *out, void *states, uint64_t state_slots,
                 const int32_t *slots_in, const int32_t *slots_out, const int32_t *starts, uint32_t rows, uint32_t seqs,
                 void *stream);

/* --------------------------------------------------------- state space --
 * Every channel has a state h [state_dim], and each token, in order, does
 *   s = softplus(dt + dt_bias);  h[n] <- e^(s a[n]) h[n] + s x b[n]
 *   out = (sum_n c[n] h[n] + skip x) (z / (1 + e^-z))
 * with b and c of the channel's group (channel / (channels / groups)). State and sums
 * are f32. */
typedef struct rl_scan rl_scan;

/* a [channels][state_dim] (negative in use), skip and dt_bias [channels] (or NULL:
 * zeros) f32 on the host, copied. state_dim 4 to 256, a multiple of 4; channels a
 * multiple of groups, at most 2^20. Workspace for calls of up to max_rows tokens in up to
 * max_seqs sequences, beside the copies of a, skip and dt_bias: at most 37 MB and four
 * states, each group's channels rounded up to whole workgroups (16 to 256 of them). */
int rl_scan_create(int device, uint32_t max_rows, uint32_t max_seqs, uint32_t channels, uint32_t groups,
                   uint32_t state_dim, const float *a, const float *skip, const float *dt_bias, rl_scan **out);
void rl_scan_destroy(rl_scan *scan);

/* x, dt, z, out [rows][1][channels] and b, c [rows][groups][state_dim] of one type; z NULL
 * leaves the last factor out, softplus 0 takes s = dt + dt_bias. out may be x, dt or z
 * itself (same data and strides), or must not overlap an input. states f32 [state_slots][channels]
 * [state_dim], slots_in, slots_out and starts as in rl_delta_rows. most_rows bounds the
 * rows of any one sequence (0: as many as the call has); it may be any number, since it
 * only picks the form that is used for all of them: one token after the other, or long
 * sequences in pieces side by side. Both are as exact as f32 sums, but do not give the
 * same bits. With softplus the lowest values of dt, and -infinity, are steps of 0, which
 * leave the state as it is. Another infinity, also one that a product or sum overflows
 * to, may read as NaN. Rows from starts[seqs] on are not written. */
int rl_scan_rows(rl_scan *scan, const rl_heads *x, const rl_heads *dt, const rl_heads *z, const rl_heads *b,
                 const rl_heads *c, const rl_heads *out, float *states, uint64_t state_slots, const int32_t *slots_in,
                 const int32_t *slots_out, const int32_t *starts, uint32_t rows, uint32_t seqs, int softplus,
                 uint32_t most_rows, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* RL_MIXERS_H */
