/* libflint: causal attention over packed sequences of different lengths, with
 * grouped heads, forward and backward.
 *
 * No counterpart in the reference's ABI (its attention takes equal lengths):
 * additive entry points.
 *
 * The sequences lie one after another in the token rows: sequence s holds rows
 * offsets[s] .. offsets[s + 1] - 1 (offsets: sequences + 1 int32 values in
 * device memory that do not decrease; equal neighbours are an empty sequence).
 * Token t of a sequence sees its sequence's tokens up to itself. Rows before
 * offsets[0] and from offsets[sequences] on belong to no sequence: they are not
 * read into any result, and their rows of every output stay as they were.
 * Offsets outside 0 .. tokens are taken as the nearer end; offsets that decrease
 * may leave any row of the outputs as it was, and lead to none outside them.
 *
 * q and o hold heads x head_width FP16 values a token, k and v kv_heads x
 * head_width; query head h reads head h / (heads / kv_heads) of k and v. Rows
 * lie q_stride, kv_stride and o_stride values apart, so q, k and v can be the
 * column slices of one projection. lse holds [heads][tokens] FP32 values.
 *
 * A non-finite value in a sequence's q, k or v may reach every row of that
 * sequence, and no other sequence. */
#ifndef FLINT_FLINT_PACKED_H
#define FLINT_FLINT_PACKED_H

#include "flint/flint.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct {
    size_t tokens;      /* rows of q, k, v, o and their gradients, up to 2^26 */
    size_t sequences;   /* up to 2^20 */
    size_t heads;       /* of q and o, up to 1,024 */
    size_t kv_heads;    /* of k and v; divides heads */
    size_t head_width;  /* 64 or 128 */
    size_t q_stride;    /* values from a row to the next of q and dq; a multiple of 8 */
    size_t kv_stride;   /* of k, v, dk and dv */
    size_t o_stride;    /* of o and dout */
} flint_packed_shape;

/* The plan lists the batch's blocks of queries, longest first. It depends on
 * offsets, tokens and sequences only: one plan serves every layer of a batch,
 * forward and backward. flint_attention_packed_plan writes it on the stream,
 * with no host synchronisation; plan and offsets are 16-byte aligned device
 * memory. */
FLINT_API flint_status flint_attention_packed_plan_bytes(const flint_packed_shape* shape,
                                                         size_t* bytes);
FLINT_API flint_status flint_attention_packed_plan(void* plan, const void* offsets,
                                                   const flint_packed_shape* shape,
                                                   flint_stream stream);

/* o[t] = sum over visible t' of softmax(scale q[t] k^T)[t'] v[t'] (RN16 of an
 * FP32 result; probabilities enter the product with v as FP16), and lse[t] =
 * log(sum over visible t' of exp(scale q[t] . k[t'])). plan must be the one of
 * this shape's tokens and sequences. scale is up to 2^64 in size. Scores past
 * 2^25 in size, where FP32 is 4 apart, may give a row NaN; and lse is an FP32
 * value, which leaves the backward pass's probabilities |lse| 2^-23 of themselves
 * off. */
FLINT_API flint_status flint_attention_packed_forward(void* o, void* lse, const void* q,
                                                      const void* k, const void* v,
                                                      const void* plan,
                                                      const flint_packed_shape* shape, float scale,
                                                      flint_stream stream);

/* dq, dk, dv: the gradients of sum(dout * o) for the o and lse that
 * flint_attention_packed_forward returned with this q, k, v, plan and scale; dk
 * and dv sum over the query heads that share a head. RN16 of FP32 results; P and
 * dS = P (dout v^T - D) enter the products as FP16, 2^8 times as large (as they
 * are where that overflows; where dS itself passes 65,504, the gradients that take
 * it are not finite). D = dout . o is that of the FP16 o; for dk it is put right by
 * the sum of dS, which is 0 otherwise. Deterministic (fixed
 * summation order, no atomics). dq, dk and dv may be column slices of one
 * tensor; they overlap no input. */
FLINT_API flint_status flint_attention_packed_backward_workspace(const flint_packed_shape* shape,
                                                                 size_t* bytes);
FLINT_API flint_status flint_attention_packed_backward(
    void* dq, void* dk, void* dv, const void* dout, const void* q, const void* k, const void* v,
    const void* o, const void* lse, const void* plan, const flint_packed_shape* shape, float scale,
    void* workspace, size_t workspace_bytes, flint_stream stream);

#ifdef __cplusplus
}
#endif

#endif /* FLINT_FLINT_PACKED_H */
