/*
 * mfh_beams.h — beam search's selection on MI355X (gfx950): the best
 * continuations of each group's beams over the vocabulary, and the beams'
 * histories in their new order.
 *
 * A step of a beam search over a paged cache (mfh_attention.h) selects here,
 * brings block tables into the same order with mfh_page_fork, whose parents
 * are this call's, and copies the pages that it lists.
 *
 * Conventions are those of mfh.h: device pointers, dtype wire codes, a stream
 * per call, MFH_OK or a negative code with mfh_last_error.  Calls are
 * asynchronous, allocate nothing and may be captured into a graph; descriptors
 * are read during the call only.
 */
#ifndef MFH_BEAMS_H
#define MFH_BEAMS_H

#include "mfh.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct {
    uint8_t dtype;        /* of the logits: Float32, Float16 or BFloat16 */
    uint8_t reserved[3];
    int32_t beams;        /* of a group, 1..256 */
    int32_t picks;        /* continuations wanted per group, 1..64 */
    int32_t vocab;        /* tokens, 1..2^24 */
    int32_t end_token;    /* the token that ends a beam, or -1 */
    int32_t reserved2;
    int64_t logits_stride;  /* of a row in elements; 0: vocab */
    int64_t history_stride; /* of a row in tokens; it holds that many */
} mfh_beam_shape;

/* Beam b of group g is row g*beams + b, with its score so far and the logits
 * that follow it.  Token t continues it with the score
 *
 *   scores[row] + logits[row][t] - log(sum over u of exp(logits[row][u]))
 *
 * and the `picks` best of a group's beams * vocab continuations become rows
 * g*picks + i of the results, best first: scores_out, tokens, and parents (the
 * row number of the beam each continues).  Continuations of equal score come
 * in the order of their beams, and those of one beam in the order of their
 * logits and then of their tokens.  Scores are compared before they are
 * rounded to f32; one below its range becomes -inf there, and keeps its token
 * and parent.
 *
 * A continuation whose score is -inf or NaN is none, nor are those of a beam
 * one of whose logits, or whose score, is NaN or +inf.  Where a group has
 * fewer than `picks`, the rest get the score -inf, token -1 and parent -1.
 *
 * ended, if not NULL, marks beams (any value but 0) that have ended: their
 * logits do not matter, and they continue only with end_token, at their score
 * as it is.  ended_out, if not NULL, marks the results that have ended, by
 * end_token or before; it may be there without `ended`.
 *
 * history, if not NULL, holds the tokens of each row so far, known[g] of
 * them in group g ([rows][history_stride]); history_out ([groups * picks]
 * [history_stride]) gets the parent's with the new token behind them.  Tokens
 * that do not fit the stride are not written, nor is the row of a result
 * without parent; what stands behind stays as it is.
 *
 * scores_out, ended_out and history_out are other buffers than scores, ended
 * and history.  The workspace (any 16-byte aligned device memory, free for
 * other use once the call's work is done) has to be as large as
 * mfh_beam_select_workspace says; what it says for more groups, beams, picks or
 * tokens does too. */
int mfh_beam_select(const mfh_beam_shape* shape, int32_t groups, const void* logits, const float* scores,
                    const uint8_t* ended, float* scores_out, int32_t* tokens, int32_t* parents, uint8_t* ended_out,
                    const int32_t* history, const int32_t* known, int32_t* history_out, void* workspace,
                    size_t workspace_bytes, void* stream);
int mfh_beam_select_workspace(const mfh_beam_shape* shape, int32_t groups, size_t* bytes);

#ifdef __cplusplus
}
#endif
#endif /* MFH_BEAMS_H */
