/* libflint: attention of new tokens over a paged cache of keys and values,
 * for generation (one new token a sequence) and for prompts taken in chunks.
 *
 * No counterpart in the reference's ABI: additive entry points.
 *
 * k_pages and v_pages hold [pages][kv_heads][page_size][head_width] FP16
 * values. Row s of table (sequences x max_pages int32) lists the pages of
 * sequence s: its position p lies in page table[s][p / page_size], row
 * p % page_size. cached[s] (int32) positions are in the cache before the call;
 * the sequence's new tokens are rows offsets[s] .. offsets[s + 1] - 1 of q, k, v
 * and o (offsets: sequences + 1 int32 values that do not decrease), at positions
 * cached[s], cached[s] + 1, ... The call
 *   - attends: a new token sees the cached positions and the sequence's new
 *     tokens up to itself;
 *   - stores the new tokens' rows of k and v into their pages, for later calls
 *     (cached itself is the caller's to advance).
 * q and o hold heads x head_width values a token, k and v kv_heads x
 * head_width; query head h reads head h / (heads / kv_heads). Rows lie
 * q_stride, kv_stride and o_stride values apart.
 *
 * Lengths and tables live on the device, so a captured call replays with the
 * values they hold then. None of them can lead outside the buffers:
 *   - a table entry outside 0 .. pages - 1 is no page: its cached positions are
 *     not seen, and new rows that would go there are not stored (they are still
 *     seen by this call's tokens);
 *   - positions past max_pages x page_size have no page either; cached[s] is
 *     taken into 0 .. max_pages x page_size, offsets into 0 .. tokens (where
 *     they decrease, any row of o may hold anything);
 *   - new tokens of a sequence past max_new are ignored, their rows of o left.
 * Rows of o outside every sequence stay as they were. Pages may be shared by
 * sequences as long as no call stores into a row that another sequence of the
 * call reads. Cache rows that hold no position (past a sequence's end, or of
 * no sequence) are not read into any result, whatever they hold. A non-finite
 * value in a sequence's q, k or v, or in its cached positions, may reach every
 * row of that sequence, and no other sequence. */
#ifndef FLINT_FLINT_PAGED_H
#define FLINT_FLINT_PAGED_H

#include "flint/flint.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct {
    size_t tokens;      /* rows of q, k, v and o, up to 2^20; tokens x heads up to 2^25 */
    size_t sequences;   /* up to 65,535; sequences x kv_heads up to 2^22 */
    size_t max_new;     /* new tokens a sequence has at most */
    size_t heads;       /* of q and o, up to 1,024 */
    size_t kv_heads;    /* of k, v and the pages; divides heads */
    size_t head_width;  /* 64 or 128 */
    size_t q_stride;    /* values from a row to the next; multiples of 8 */
    size_t kv_stride;
    size_t o_stride;
    size_t pages;       /* of k_pages and v_pages, up to 2^31 - 1, and 2^46 values in all */
    size_t page_size;   /* positions a page: a multiple of 8 up to 65,536 */
    size_t max_pages;   /* columns of table; max_pages x page_size up to 2^30 */
} flint_paged_shape;

FLINT_API flint_status flint_attention_paged_workspace(const flint_paged_shape* shape,
                                                       size_t* bytes);

/* o[t] = sum over visible positions of softmax(scale q[t] k^T) v, RN16 of an
 * FP32 result; probabilities enter the product with v as FP16. scale is up to 2^64 in size; scores past 2^25 in size, where FP32
 * is 4 apart, may give a row NaN. The workspace needs no preparation and keeps nothing between
 * calls. */
FLINT_API flint_status flint_attention_paged(void* o, void* k_pages, void* v_pages, const void* q,
                                             const void* k, const void* v, const void* offsets,
                                             const void* cached, const void* table,
                                             const flint_paged_shape* shape, float scale,
                                             void* workspace, size_t workspace_bytes,
                                             flint_stream stream);

#ifdef __cplusplus
}
#endif

#endif /* FLINT_FLINT_PAGED_H */
