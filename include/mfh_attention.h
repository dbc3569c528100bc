/*
 * mfh_attention.h — serving over a paged key-value cache on MI355X (gfx950):
 * block tables and slot maps, rotary positions with the cache's writes, and
 * attention over pages for one new token per request (decode) or many
 * (prefill).
 *
 * The reference plans paged key-value state on the host (runtime/paged_plan.go:41,
 * runtime/paged_executor.go:15) and leaves the device's part to a backend; these
 * entry points are that part.  A step of a decoder runs them in this order:
 *
 *   mfh_page_plan         lengths before and after -> pages, slots, positions
 *   mfh_rotary_append     q, k turned by position; k, v written to their slots
 *   mfh_paged_prefill     or, where every request has one new token,
 *   mfh_paged_decode      attention over what the cache now holds
 *
 * Conventions are those of mfh.h: device pointers, dtype wire codes, a stream
 * per call, MFH_OK or a negative code with mfh_last_error.  Every call is
 * asynchronous, allocates nothing and may be captured into a graph; what
 * differs from step to step (lengths, tables, slots) is read on the device.
 * Descriptors are read during the call only.
 *
 * Values on the device cannot be checked by the host: page numbers outside the
 * cache, slots outside it and lengths past a table's row are never followed.
 * Such a page's tokens count as masked, such a slot is not written, and a
 * length counts as that of the whole row, or as 2^30 where that is less.
 */
#ifndef MFH_ATTENTION_H
#define MFH_ATTENTION_H

#include "mfh.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- the cache ------------------------------------------------------------ */

/* Keys and values live in two buffers of one layout.  Element (page, token of
 * the page, head, d) stands at page*page_stride + token*token_stride +
 * head*head_stride + d (strides in elements, not negative); a page's tokens
 * and heads span less than 2 GiB.  Token t of a request is token t % page_size
 * of page table[request][t / page_size], and its slot is
 * page*page_size + t % page_size. */
typedef struct {
    uint8_t dtype;       /* Float16, BFloat16 or Float8E4M3 */
    uint8_t reserved[3];
    int32_t page_size;   /* tokens of a page, any positive number */
    int32_t kv_heads;
    int32_t head_dim;    /* a multiple of 8 (Float8E4M3: of 16), up to 256 */
    int64_t pages;
    int64_t page_stride;
    int64_t token_stride;
    int64_t head_stride;
    float k_scale;       /* Float8E4M3: a key is its code times k_scale, */
    float v_scale;       /* a value its code times v_scale; else both are 1 */
} mfh_kv_cache;

/* ---- block tables and slot maps ------------------------------------------- */

/* One step of the page allocator.  Request r goes from before[r] cached tokens
 * to after[r]; a larger number asks for pages and slots, a smaller one returns
 * pages (0: the request has ended).  Free pages wait in a ring: `ring` holds
 * ring_size page numbers, ring_state[0] (head) and ring_state[1] (tail) count
 * the pages ever taken and ever returned, free pages are ring[i % ring_size]
 * for head <= i < tail.  In the order of requests, pages are taken from the
 * head and written to table[r] behind the pages that r has; returned pages go
 * to the tail and can be taken from the next call on.  The ring has room for
 * every page of the cache.  ring_state_out receives the new head and tail and
 * is another buffer than ring_state.
 *
 * New tokens are numbered request after request: those of r are starts[r] ..
 * starts[r+1]-1, each with its position in the request and its slot.  Numbers
 * past the last one up to `tokens` (a captured step's padding) get position -1
 * and slot -1.
 *
 * status[r]: 0 done; 1 no pages were left (each later request that needs pages
 * is refused too); 2 a length is negative or needs more than table_width
 * pages; 3 its tokens do not fit into `tokens`.  A refused request takes and
 * returns nothing, its tokens get the slot -1 and lengths[r] is before[r]
 * (0 where that is negative); of the others lengths[r] is after[r].
 *
 * table is [requests][table_stride] with table_width entries in use; entries
 * behind a request's pages keep what they held.  lengths is another buffer than
 * before and after, or, in a call of at most 512 tokens, may be one of them.
 * starts has requests + 1 entries.  requests >= 0, 0 <= tokens <= 2^30,
 * 0 < ring_size <= 2^30. */
int mfh_page_plan(const int32_t* before, const int32_t* after, int32_t requests, int32_t page_size,
                  int32_t* table, int64_t table_stride, int32_t table_width,
                  int32_t* ring, int64_t ring_size, const int64_t* ring_state, int64_t* ring_state_out,
                  int64_t* slots, int32_t* positions, int64_t tokens, int32_t* starts, int32_t* lengths,
                  int32_t* status, void* stream);

/* ---- rotary positions ------------------------------------------------------ */

/* How a model's positions outgrow those it was trained on. */
#define MFH_ROTARY_PLAIN 0  /* base^(-2i/dim) */
#define MFH_ROTARY_LINEAR 1 /* positions divided by factor */
#define MFH_ROTARY_BASE 2   /* base * factor^(dim/(dim-2)): the slowest pair as under LINEAR, the fastest as under PLAIN */
#define MFH_ROTARY_BANDS 3  /* by turns over original_length: above high PLAIN, below low LINEAR, between them mixed in proportion */

/* Writes the rotary_dim / 2 frequencies (radians per position) to host memory.
 * BANDS: pair i turns n = original_length * f / (2 pi) times over the original
 * length; its frequency is f * (s + (1 - s) / factor) with
 * s = clamp((n - low) / (high - low), 0, 1). */
int mfh_rotary_frequencies(double* out, int32_t rotary_dim, double base, int32_t scaling, double factor,
                           double original_length, double low, double high);

typedef struct {
    uint8_t dtype;       /* of q, k and v: Float32, Float16 or BFloat16 */
    uint8_t interleaved; /* pair i is elements 2i, 2i+1; else i, i + rotary_dim/2 */
    uint8_t inverse;     /* turn back: the gradient of the turn */
    uint8_t reserved;
    int32_t q_heads;
    int32_t kv_heads;
    int32_t head_dim;    /* even */
    int32_t rotary_dim;  /* even, 0..head_dim; the elements behind it are copied */
    float factor;        /* multiplies cosine and sine (1, or a long context's attention factor) */
    int64_t q_token_stride, q_head_stride;         /* strides in elements; a pair of zeros: dense [tokens][heads][dim] */
    int64_t q_out_token_stride, q_out_head_stride;
    int64_t k_token_stride, k_head_stride;
    int64_t k_out_token_stride, k_out_head_stride;
    int64_t v_token_stride, v_head_stride;
} mfh_rotary_shape;

/* Turns pair (a, b) of token t into (a c - b s, b c + a s), c and s the cosine
 * and sine of positions[t] * frequencies[i] times factor, in f32 from a phase
 * reduced in f64.  q and k are [tokens][heads][head_dim]; either may be NULL
 * with its result.  A result may be its own input (same strides).
 * frequencies: rotary_dim / 2 f64 values in device memory. */
int mfh_rotary(const mfh_rotary_shape* shape, int64_t tokens, const void* q, void* q_out, const void* k,
               void* k_out, const int32_t* positions, const double* frequencies, void* stream);

/* mfh_rotary of q and k with k and v written to their slots of the cache, in
 * the cache's dtype: that of the shape, or Float8E4M3, where a value is
 * multiplied by its scale's reciprocal, limited to +-448 and rounded to the
 * nearest code (ties to even; a NaN stays NaN).  A token whose slot is outside the cache is not written.
 * Slots of one call differ.  The k_out strides are not used; q may be NULL
 * with q_out.  `inverse` is refused. */
int mfh_rotary_append(const mfh_rotary_shape* shape, const mfh_kv_cache* cache, int64_t tokens, const void* q,
                      void* q_out, const void* k, const void* v, const int32_t* positions, const int64_t* slots,
                      const double* frequencies, void* k_cache, void* v_cache, void* stream);

/* ---- attention --------------------------------------------------------------- */

typedef struct {
    uint8_t dtype;      /* of q and out: Float16 or BFloat16; the cache has the same or Float8E4M3 */
    uint8_t reserved[3];
    int32_t q_heads;    /* group * kv_heads: heads h*group .. h*group + group-1 read key-value head h */
    float scale;        /* of q.k, before the cap */
    float softcap;      /* > 0: a score x becomes softcap * tanh(x / softcap) */
    int32_t window;     /* > 0: a token sees the last `window` positions, its own among them */
    int64_t q_token_stride, q_head_stride;     /* strides in elements; both 0: dense [tokens][heads][dim] */
    int64_t out_token_stride, out_head_stride; /* the same */
} mfh_attention_shape;

/* Attention of one new token per request, whose key and value are already in
 * the cache: out[r][h] = sum_j p_j v_j / sum_j p_j over the positions
 * j < lengths[r] (of the window), p_j = exp(score_j - max).  slopes, if not
 * NULL, holds one f32 per query head, and a score loses slope * distance.
 * lse, if not NULL, receives log(sum exp(score)) as f32 [requests][q_heads].
 * A request of length 0 gives zeros and -inf.  What stands behind a request's
 * length in its last page does not matter, NaN included.
 *
 * Long contexts are split over workgroups; their parts meet in `workspace`
 * (mfh_paged_decode_workspace bytes, any 16-byte aligned device memory, free
 * for other use once the call's work is done; with less, or none, the call
 * does not split).  longest is the caller's upper bound of the lengths: it
 * decides the split, and with it the order of the sums, nothing else. */
int mfh_paged_decode(const mfh_attention_shape* shape, const mfh_kv_cache* cache, int32_t requests, const void* q,
                     const void* k_cache, const void* v_cache, const int32_t* table, int64_t table_stride,
                     int32_t table_width, const int32_t* lengths, int64_t longest, const float* slopes, void* out,
                     float* lse, void* workspace, size_t workspace_bytes, void* stream);
int mfh_paged_decode_workspace(const mfh_attention_shape* shape, const mfh_kv_cache* cache, int32_t requests,
                               int64_t longest, size_t* bytes);

/* Attention of each request's new tokens, whose keys and values are already in
 * the cache.  Tokens starts[r] .. starts[r+1]-1 of q and out are the last ones
 * of request r, at positions lengths[r] - n .. lengths[r] - 1; each sees the
 * positions up to its own (of the window), and with prefix, if not NULL, the
 * first prefix[r] positions of its request too, later ones among them.  slopes
 * as above, by the distance either way.  A token that sees nothing gives zeros
 * and -inf.  Masked positions do not matter, whatever they hold.
 *
 * tokens is the number of rows of q and out (starts past it are cut off);
 * most_fresh is an upper bound of the requests' new tokens, and a request's
 * tokens past it are not computed.  longest is as above, and so is the workspace,
 * but that with less of it the call has fewer parts. */
int mfh_paged_prefill(const mfh_attention_shape* shape, const mfh_kv_cache* cache, int32_t requests, int64_t tokens,
                      int64_t most_fresh, const void* q, const void* k_cache, const void* v_cache,
                      const int32_t* table, int64_t table_stride, int32_t table_width, const int32_t* starts,
                      const int32_t* lengths, int64_t longest, const int32_t* prefix, const float* slopes, void* out,
                      float* lse, void* workspace, size_t workspace_bytes, void* stream);
int mfh_paged_prefill_workspace(const mfh_attention_shape* shape, const mfh_kv_cache* cache, int32_t requests,
                                int64_t tokens, int64_t most_fresh, int64_t longest, size_t* bytes);

#ifdef __cplusplus
}
#endif
#endif /* MFH_ATTENTION_H */
