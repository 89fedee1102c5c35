/*
 * tilegen_b200_paged.h -- C ABI of the paged-attention operators of libtilegen_b200.so:
 * rotary positions, appending to a paged key/value cache, and attention of a batch of
 * sequences that share a prefix.
 *
 * The calls follow the native API of tilegen_b200.h: asynchronous on the given stream, no
 * internal synchronisation, no allocation (the attention takes a caller's workspace),
 * TG_OK or a negative TG_E* status with the message in tg_last_error_string().  All
 * pointers are device pointers unless stated otherwise; the descriptors themselves are
 * host memory and are read before the call returns.
 *
 * Which pages hold a sequence's keys and values is a CSR pattern: a tg_csr whose rows are
 * the sequences, whose columns are the cache's pages (cols = number of pages, data
 * unused) and whose row b lists the pages of sequence b in the order of its tokens.
 *
 * Index arrays are the caller's promise, as for the sparse calls: page numbers inside the
 * cache, lengths inside the listed pages.  Without TG_FLAG_BOUNDS_CHECK an entry that
 * breaks it never makes a kernel read or write outside the given arrays (a write to a
 * page that does not exist is dropped, a read gives zeros, a length is cut to the listed
 * pages); with the flag the arrays are checked first, synchronously, and the call returns
 * TG_EBOUNDS without having run.
 */
#ifndef TILEGEN_B200_PAGED_H
#define TILEGEN_B200_PAGED_H

#include "tilegen_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* flags of these calls, beside TG_FLAG_BOUNDS_CHECK */
#define TG_FLAG_CAUSAL 16u       /* attention: a query sees no key after its own token */
#define TG_FLAG_ROPE_INVERSE 32u /* tg_rope_*: the transpose (the gradient of the rotation) */

#define TG_ROPE_HALF 0        /* element i turns with element i + rot_dim/2 */
#define TG_ROPE_INTERLEAVED 1 /* element 2i turns with element 2i + 1 */

/* A rotation: pair i of a head's first rot_dim elements turns by position * freq[i]
 * radians and is multiplied by scale; the other elements are copied. */
typedef struct tg_rope {
    const double* freq; /* rot_dim / 2 values */
    int32_t rot_dim;    /* even, 0 .. head dim */
    int32_t layout;     /* TG_ROPE_* */
    double scale;
} tg_rope;

/* tokens x heads rows of `dim` consecutive elements, strides in elements. */
typedef struct tg_rows {
    void* data;
    int64_t token_stride;
    int64_t head_stride;
} tg_rows;

/* Keys and values of `heads` heads in pages of page_size tokens, strides in elements; a
 * head's `dim` elements are consecutive. */
typedef struct tg_paged_kv {
    void* k;
    void* v;
    int64_t pages;
    int64_t page_size;
    int32_t heads;
    int32_t dim;
    int64_t k_page_stride, k_slot_stride, k_head_stride;
    int64_t v_page_stride, v_slot_stride, v_head_stride;
} tg_paged_kv;

/* y = rotation of x at the tokens' positions (int64), or with TG_FLAG_ROPE_INVERSE the
 * gradient with respect to x for the gradient x of the output.  y may be x itself. */
TG_API int tg_rope_f32(const tg_rope* r, const tg_rows* x, const tg_rows* y, int64_t tokens, int32_t heads,
                       int32_t dim, const int64_t* positions, uint32_t flags, tg_stream_t stream);
TG_API int tg_rope_f16(const tg_rope* r, const tg_rows* x, const tg_rows* y, int64_t tokens, int32_t heads,
                       int32_t dim, const int64_t* positions, uint32_t flags, tg_stream_t stream);
TG_API int tg_rope_bf16(const tg_rope* r, const tg_rows* x, const tg_rows* y, int64_t tokens, int32_t heads,
                        int32_t dim, const int64_t* positions, uint32_t flags, tg_stream_t stream);

/* New tokens of a batch.  Sequence b brings the tokens q_indptr[b] .. q_indptr[b+1]
 * (q_indptr NULL: token b alone, tokens == pages->rows) and is seq_len[b] tokens long
 * after them, so its i-th new token is token a = seq_len[b] - n + i of its own pages.  k and
 * v are written there; k is rotated by r at position positions[t], or position_base + a
 * where positions is NULL.  With q (q_heads heads) not NULL, q_out receives q rotated at
 * the same position (q_out may be q).  r NULL: nothing turns.  Two new tokens must not
 * share a slot. */
typedef struct tg_kv_append_args {
    const tg_paged_kv* cache;
    const tg_csr* pages;
    const int64_t* seq_len;
    int64_t tokens;
    const int64_t* q_indptr;
    tg_rows k, v;
    const tg_rope* rope;
    const tg_rows* q;
    const tg_rows* q_out;
    int32_t q_heads;
    int64_t position_base;
    const int64_t* positions;
    uint32_t flags;
} tg_kv_append_args;
TG_API int tg_kv_append_f32(const tg_kv_append_args* a, tg_stream_t stream);
TG_API int tg_kv_append_f16(const tg_kv_append_args* a, tg_stream_t stream);
TG_API int tg_kv_append_bf16(const tg_kv_append_args* a, tg_stream_t stream);

/* The norm of a head x of `dim` elements: x / sqrt(mean(x^2) + eps) * (offset + weight[i]), or
 * without that factor where weight is NULL.  The mean and all sums are 32-bit. */
typedef struct tg_head_norm {
    const void* weight; /* dim values, or NULL */
    int32_t weight_f32; /* the weight is float, else of the rows' type */
    double eps;         /* >= 0 */
    double offset;
} tg_head_norm;

/* q_out = rotation of the normed q at the tokens' positions, and the same for k, in one pass.  An
 * output may be its input.  A norm NULL: that tensor is only rotated; rope NULL: nothing turns and
 * positions are not read; a number of heads 0: that tensor is not there.  dim at most 256. */
typedef struct tg_norm_rope_args {
    int64_t tokens;
    int32_t dim;
    int32_t q_heads, k_heads;
    tg_rows q, k, q_out, k_out;
    const tg_head_norm* q_norm;
    const tg_head_norm* k_norm;
    const tg_rope* rope;
    const int64_t* positions;
    uint32_t flags; /* 0 */
} tg_norm_rope_args;
TG_API int tg_norm_rope_f32(const tg_norm_rope_args* a, tg_stream_t stream);
TG_API int tg_norm_rope_f16(const tg_norm_rope_args* a, tg_stream_t stream);
TG_API int tg_norm_rope_bf16(const tg_norm_rope_args* a, tg_stream_t stream);

/* Its gradient: for the gradients dq_out and dk_out of the outputs, those of the inputs (dq, dk;
 * each may be dq_out, dk_out or the input itself) and of the weights (of the weight's type, summed
 * over all tokens and heads of the tensor in 32 bits and in a fixed order; NULL: not wanted). */
typedef struct tg_norm_rope_grad_args {
    int64_t tokens;
    int32_t dim;
    int32_t q_heads, k_heads;
    tg_rows q, k, dq_out, dk_out, dq, dk;
    const tg_head_norm* q_norm;
    const tg_head_norm* k_norm;
    void* dq_weight;
    void* dk_weight;
    const tg_rope* rope;
    const int64_t* positions;
    uint32_t flags; /* 0 */
} tg_norm_rope_grad_args;
/* Bytes of its workspace; it serves every call with heads no longer and as many tokens or fewer. */
TG_API size_t tg_norm_rope_backward_workspace_bytes(const tg_norm_rope_grad_args* a);
TG_API int tg_norm_rope_backward_f32(const tg_norm_rope_grad_args* a, void* workspace, size_t workspace_bytes,
                                     tg_stream_t stream);
TG_API int tg_norm_rope_backward_f16(const tg_norm_rope_grad_args* a, void* workspace, size_t workspace_bytes,
                                     tg_stream_t stream);
TG_API int tg_norm_rope_backward_bf16(const tg_norm_rope_grad_args* a, void* workspace, size_t workspace_bytes,
                                      tg_stream_t stream);

/* tg_kv_append_* with norms of q and k before the rotation (NULL: none).  dim at most 256. */
TG_API int tg_kv_append_normed_f32(const tg_kv_append_args* a, const tg_head_norm* q_norm, const tg_head_norm* k_norm,
                                   tg_stream_t stream);
TG_API int tg_kv_append_normed_f16(const tg_kv_append_args* a, const tg_head_norm* q_norm, const tg_head_norm* k_norm,
                                   tg_stream_t stream);
TG_API int tg_kv_append_normed_bf16(const tg_kv_append_args* a, const tg_head_norm* q_norm, const tg_head_norm* k_norm,
                                    tg_stream_t stream);

/* out = softmax(scale * q k^T) v for the queries of a batch (tokens by q_indptr as above).
 * The keys of sequence b are the prefix_len tokens of the prefix pages, shared by the whole
 * batch, followed by the seq_len[b] tokens of its own pages.  Query head j uses key head
 * j / (q_heads / cache->heads).  With TG_FLAG_CAUSAL the i-th of the n queries of sequence b
 * sees the first prefix_len + seq_len[b] - n + i + 1 keys, without it all; a query that sees
 * none gives zeros.  What lies in the cache beyond what a query sees (NaN and infinities
 * included) has no effect on it.  lse, where not NULL, receives log(sum(exp(scale * q k^T)))
 * of each (token, head), -inf where nothing is seen.
 *
 * The prefix is fetched once for every 256 rows (tokens times the query heads of a key head)
 * where dim is 64 or 128 and rows are more than 32, else once for every 16 or 32; those
 * fetches meet in L2.  Products are summed and the softmax is taken in 32 bits.  The weights
 * exp(...) are rounded to the values' type for their product with them: relative errors of
 * half an ulp that average out over the keys, together with the output's own rounding about
 * 1.4 times the error of that alone.
 *
 * max_seq_len bounds the entries of seq_len; a longer one counts as max_seq_len.  max_q_len
 * (not 0) bounds the tokens of one sequence: the first max_q_len see what they see without
 * the bound, those after them, and tokens that no sequence holds, see nothing.  Dim 64, 96,
 * 128 or 256; all rows 16-byte aligned and all strides multiples of 8 elements, but those of
 * dimensions of one, which are not read.  out may not share memory with q. */
typedef struct tg_prefix_attention_args {
    const tg_paged_kv* cache;
    const tg_csr* pages;
    const int64_t* seq_len;
    int64_t max_seq_len;
    const int64_t* prefix_pages; /* n_prefix_pages page numbers */
    int64_t n_prefix_pages;
    int64_t prefix_len;
    int64_t tokens;
    const int64_t* q_indptr;
    int64_t max_q_len;
    int32_t q_heads;
    tg_rows q, out;
    float* lse; /* [tokens, q_heads] or NULL */
    double scale; /* > 0 */
    uint32_t flags;
} tg_prefix_attention_args;
/* Bytes of a workspace to keep: enough for a call with these arguments and for any with the
 * same head sizes and at most as many tokens, sequences, listed pages and prefix tokens and
 * no larger max_seq_len and max_q_len (pointers are not read); 0 also where the arguments are
 * not valid.  It stays below 1.1 GiB and three parts of each row together. */
TG_API size_t tg_prefix_attention_workspace_bytes(const tg_prefix_attention_args* a);
/* What a call with these very arguments takes, at most the former: for one that allocates.
 * A smaller call may take more. */
TG_API size_t tg_prefix_attention_needed_bytes(const tg_prefix_attention_args* a);
TG_API int tg_prefix_attention_f16(const tg_prefix_attention_args* a, void* workspace, size_t workspace_bytes,
                                   tg_stream_t stream);
TG_API int tg_prefix_attention_bf16(const tg_prefix_attention_args* a, void* workspace, size_t workspace_bytes,
                                    tg_stream_t stream);

/* A 32-bit number for each cached key, strides in elements. */
typedef struct tg_paged_mass {
    float* data;
    int64_t page_stride, slot_stride, head_stride;
} tg_paged_mass;

/* The attention weight that the keys of the sequences' own pages gather from the queries of a batch:
 *   mass[key] = decay * mass[key] + sum of exp(scale * q k - lse)
 * over the rows (new token, query head of the key's head) that see the key, with q, lse
 * ([tokens, q_heads]), scale and TG_FLAG_CAUSAL as given to and returned by tg_prefix_attention_*:
 * with a prefix, lse holds the prefix's share too, and the own keys get theirs.  Tokens and lengths
 * as there; tokens past the first max_q_len of a sequence add nothing, nor does a row whose lse is
 * -inf.  With TG_FLAG_CAUSAL the last n keys are those of the n new tokens: what their slots held
 * before is not read.  Nor is anything where decay is 0.  Every key of a sequence is written, keys
 * that no row sees with decay * mass; slots behind a sequence's length are left alone, and slots of
 * pages that do not exist dropped.  No page may be listed twice.  Scores, exponentials and sums are
 * 32-bit and the sums' order is fixed.  cache->v is not read.  Dim 64, 96, 128 or 256, q and k
 * aligned as for the attention.  A block of the kernel whose warps wait for one another longer than
 * two seconds (environment: TG_MASS_WAIT_MS) leaves NaN in the mass of all its keys. */
typedef struct tg_attention_mass_args {
    const tg_paged_kv* cache;
    const tg_csr* pages;
    const int64_t* seq_len;
    int64_t max_seq_len;
    int64_t tokens;
    const int64_t* q_indptr;
    int64_t max_q_len;
    int32_t q_heads;
    tg_rows q;
    const float* lse;
    double scale; /* > 0 */
    tg_paged_mass mass;
    double decay; /* >= 0 */
    uint32_t flags;
} tg_attention_mass_args;
/* Bytes of a workspace to keep, enough for any call of the same heads with no larger max_q_len, with or
 * without q_indptr and however many tokens (0 for few rows; never more than 80 MB). */
TG_API size_t tg_attention_mass_workspace_bytes(const tg_attention_mass_args* a);
/* What a call with these very arguments takes, at most the former. */
TG_API size_t tg_attention_mass_needed_bytes(const tg_attention_mass_args* a);
TG_API int tg_attention_mass_f16(const tg_attention_mass_args* a, void* workspace, size_t workspace_bytes,
                                 tg_stream_t stream);
TG_API int tg_attention_mass_bf16(const tg_attention_mass_args* a, void* workspace, size_t workspace_bytes,
                                  tg_stream_t stream);

/* Cuts each sequence longer than `budget` to it, in place: for each key head by itself the first
 * `first` places, the last `recent` ones and, of those between, the places with the largest mass stay
 * (equal ones from the lowest place on; NaN counts as the largest, -0 as 0).  Where the budget is
 * smaller, `recent` goes before `first`.  New places: the first ones as they were; then the chosen
 * ones, of which those that lie within the places of their number stay and the others, in the order of
 * their places, fill what is free there, from the lowest place on; then the recent ones in their
 * order.  Keys, values and mass move together; mass_out (data NULL: mass itself) receives the mass of
 * all kept keys and must not share memory with mass otherwise.  What lies behind the new length is
 * undefined, nothing else is written.  Shorter sequences stay as they are.
 *
 * seq_len_out (it may be seq_len) receives the lengths, kept[sequence][head][kept_width], where not
 * NULL, each new place's old one, -1 behind the new length; kept_width is at least the smaller of
 * budget and max_seq_len.  A sequence longer than max_seq_len counts as that long.  No page may be
 * listed twice.  Of pages that do not exist mass, keys and values read as zeros and writes are
 * dropped. */
typedef struct tg_kv_evict_args {
    const tg_paged_kv* cache;
    const tg_csr* pages;
    const int64_t* seq_len;
    int64_t max_seq_len;
    int64_t budget, first, recent;
    tg_paged_mass mass, mass_out;
    int64_t* seq_len_out;
    int32_t* kept;
    int64_t kept_width;
    uint32_t flags; /* 0 or TG_FLAG_BOUNDS_CHECK */
} tg_kv_evict_args;
/* Bytes of a workspace: enough for any call of the same budget and number of heads with no more
 * sequences and listed pages and no larger max_seq_len. */
TG_API size_t tg_kv_evict_workspace_bytes(const tg_kv_evict_args* a);
TG_API int tg_kv_evict_f32(const tg_kv_evict_args* a, void* workspace, size_t workspace_bytes, tg_stream_t stream);
TG_API int tg_kv_evict_f16(const tg_kv_evict_args* a, void* workspace, size_t workspace_bytes, tg_stream_t stream);
TG_API int tg_kv_evict_bf16(const tg_kv_evict_args* a, void* workspace, size_t workspace_bytes, tg_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* TILEGEN_B200_PAGED_H */
