/* libflint: attention of new tokens over a paged cache of keys and values held in 8
 * bits, with a scale a block of positions and head: half of flint_paged.h's bytes.
 *
 * No counterpart in the reference's ABI: additive entry points.
 *
 * Shapes, rows, lengths, tables, what is read, stored and left alone are
 * flint_attention_paged's (flint_paged.h), but for the pages: k_pages and v_pages hold
 * [pages][kv_heads][page_size][head_width] bytes, e4m3 numbers (no infinities, largest
 * 448), and k_scales and v_scales [pages][kv_heads][page_size / block] bytes. A value is
 * its number times 2^(byte - 127) of its block of `block` positions (a power of two up to
 * 128 that divides page_size). Bytes are 112 to 135 (2^-15 to 2^8; others are taken as the
 * nearer end), and values within FP16's range, which holds every one exactly.
 *
 * The call attends over the cache as it was and over the new tokens' rows as they are
 * given, in FP16; then it stores those. A block's scale becomes the least at which the
 * largest finite value of its new rows is at most 448, or stays what it was where that is
 * more and the block holds older positions of the sequence; where it grows, they are
 * rounded again. A row's values are rounded to nearest even, to the largest that fits
 * where they pass it (65,504 becomes 61,440), and non-finite ones to NaN.
 *
 * Pages may be shared by sequences as long as no call stores into a block that another
 * sequence of the call reads or stores into.
 *
 * Single tokens and chunks of prompts are best called apart (flint_paged.h): 63 tokens of
 * sequences over 1,024 to 8,192 positions and a chunk of 500 over 4,096, 32 heads on 8 of
 * 128, take 341 us in one call and 125 + 74 in two. */
#ifndef FLINT_FLINT_PAGED8_H
#define FLINT_FLINT_PAGED8_H

#include "flint/flint.h"
#include "flint/flint_paged.h"

#ifdef __cplusplus
extern "C" {
#endif

FLINT_API flint_status flint_attention_paged8_workspace(const flint_paged_shape* shape, size_t block,
                                                        size_t* bytes);

/* As flint_attention_paged, with its FP16 probabilities: o is about 1.4 times as far from the
 * exact result as storing it in FP16 alone leaves it. */
FLINT_API flint_status flint_attention_paged8(void* o, void* k_pages, void* k_scales, void* v_pages,
                                              void* v_scales, const void* q, const void* k,
                                              const void* v, const void* offsets, const void* cached,
                                              const void* table, const flint_paged_shape* shape,
                                              size_t block, float scale, void* workspace,
                                              size_t workspace_bytes, flint_stream stream);

#ifdef __cplusplus
}
#endif

#endif /* FLINT_FLINT_PAGED8_H */
