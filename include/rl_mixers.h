/*
 * rl_mixers.h — C ABI of the MI355X (gfx950) token mixers: what the layers
 * between the embedding lookup and the output head (rl_head.h) do across the
 * tokens of a sequence. Rotary positions, a paged key-value cache that is
 * quantised as it is written, attention of new tokens over that cache, and the
 * gated delta rule.
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
 * max_rows * q_heads * min(max_len / 1536 + 1, 256), at most 2^20, at least 24576.
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

#ifdef __cplusplus
}
#endif

#endif /* RL_MIXERS_H */
