/*
 * rl_drafts.h — C ABI of the verification of drafted tokens on the MI355X (gfx950):
 * how many tokens of a draft a target model's probabilities accept, and the token
 * after them, so that what comes out is distributed as the target's own draws.
 *
 * Conventions as in rl_sampler.h: status codes, rl_sampler_last_error() for the
 * message, stream-ordered calls that return before the kernels finish, one thread
 * and one stream at a time per handle. The create function allocates all a call
 * needs; calls may be captured into a graph.
 */
#ifndef RL_DRAFTS_H
#define RL_DRAFTS_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Probabilities of rows of tokens, f32 in device memory, `row_stride` elements from a
 * row to the next. With ids NULL row r has probs[r * row_stride + v] for every token v
 * of the vocabulary. Else it is a candidate list as rl_sampler_sample_rows writes it:
 * its first kept[r] entries (at most row_stride) give ids[r * row_stride + j] the
 * probability probs[r * row_stride + j], and every other token has none. A list's ids
 * are distinct. A probability that is not a positive finite number counts as none. */
typedef struct rl_probs {
    const float *probs;
    uint64_t row_stride;
    const uint32_t *ids;
    const uint32_t *kept;
} rl_probs;

typedef struct rl_drafts rl_drafts;

/* Workspace for calls of up to max_seqs sequences over `vocab` tokens: 8 bytes for
 * each 4096 tokens, or begun ones, and 4 bytes, a sequence. max_seqs at most 2^16,
 * vocab at most 2^21. */
int rl_drafts_create(int device, uint32_t max_seqs, uint32_t vocab, rl_drafts **out);
void rl_drafts_destroy(rl_drafts *drafts);

/* Sequence s has the drafted tokens drafted[starts[s] .. starts[s + 1]) (i32; starts
 * i32 [seqs + 1] rises from 0 to `drafts`). Draft j of the call has row j of `draft`,
 * the probabilities it was drawn from; `target` has one row more a sequence than it has
 * drafts: row starts[s] + s + i are the probabilities of the token at the place of its
 * draft i, the last one those of the token after all. In order, draft d with
 * probabilities p of the target and q of the draft is accepted if
 *   uniforms[j] * q(d) < p(d)
 * At the first that is not, the sequence's token is drawn from max(p - q, 0) of that
 * row; where all are accepted it is drawn from p of the last. A draw takes the first
 * token, in order of the row's entries, at which the running sum passes draws[s] times
 * the sum of all. Products and sums are f64. Where max(p - q, 0) is nowhere above zero
 * it is drawn from p, and where p is not either the token is -1.
 *
 * draft NULL: the drafts were not drawn, and q is 1 at the drafted token. draft is
 * dense where target is, and lists where target is. A drafted token outside the
 * vocabulary (of a list: that it does not hold) has p = q = 0 and is not accepted.
 * uniforms f32 [drafts] and draws f32 [seqs] in [0, 1); a draw of 1 or more or NaN
 * takes the last token that can be drawn, one below 0 the first.
 *
 * accepted i32 [seqs], which like tokens must not overlap an input: drafts accepted.
 * tokens i32 [drafts + seqs]: from starts[s] + s on the accepted ones, the drawn one and
 * -1 up to the next sequence's. */
int rl_drafts_verify(rl_drafts *drafts_handle, const rl_probs *target, const rl_probs *draft, const int32_t *drafted,
                     const int32_t *starts, const float *uniforms, const float *draws, uint32_t drafts, uint32_t seqs,
                     int32_t *accepted, int32_t *tokens, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* RL_DRAFTS_H */
