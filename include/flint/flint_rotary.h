/* libflint: rotary positions. Each head's pairs of values of q and k are turned
 * by an angle that grows with the token's position, before the attention over
 * packed sequences or over a paged cache.
 *
 * No counterpart in the reference's ABI: additive entry points.
 *
 * The first `width` values of a head turn, in width / 2 pairs (a, b): values i
 * and i + width / 2 (FLINT_ROTARY_HALVES), or 2i and 2i + 1 (FLINT_ROTARY_PAIRS).
 * At position p pair i becomes
 *   (m (a cos t - b sin t), m (a sin t + b cos t)),   t = p f_i,
 * RN16 of an FP32 result; the head's other values are copied. p f_i is formed in
 * FP64, so far positions lose nothing. */
#ifndef FLINT_FLINT_ROTARY_H
#define FLINT_FLINT_ROTARY_H

#include "flint/flint.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { FLINT_ROTARY_HALVES = 0, FLINT_ROTARY_PAIRS = 1 };

/* The frequencies f_i = base^(-2i / width), scaled for contexts longer than the
 * trained one: with r = original f_i / 2 pi turns over the trained length and
 * g = (r - low) / (high - low) taken into 0 .. 1, f_i becomes
 * f_i (g + (1 - g) / factor). Fast pairs (r >= high) keep their frequency, slow
 * ones (r <= low) are divided by factor; original = 0 divides all of them (low
 * and high are not read then), factor = 1 none. */
typedef struct {
    size_t width;     /* even, 2 to 1,024 */
    double base;      /* above 1 */
    double factor;    /* positive */
    double original;  /* trained length in positions, or 0 */
    double low;       /* turns; low < high */
    double high;
    double magnitude; /* m above; 1 leaves lengths as they are */
} flint_rotary_angles;

/* A plan holds 1 + width / 2 FP64 values: m, then f_i / 2 pi, the turns a
 * position (a caller with frequencies of its own writes these). It depends on the
 * angles alone: one plan serves every layer and call, forward and backward.
 * flint_rotary_plan writes it on the stream; 16-byte aligned device memory. */
FLINT_API flint_status flint_rotary_plan_bytes(size_t width, size_t* bytes);
FLINT_API flint_status flint_rotary_plan(void* plan, const flint_rotary_angles* angles,
                                         flint_stream stream);

typedef struct {
    size_t tokens;        /* rows, up to 2^26 */
    size_t heads;         /* of q, up to 1,024; 0: q and q_out are not read or written */
    size_t kv_heads;      /* of k, up to 1,024; 0 likewise */
    size_t head_width;    /* a multiple of 8 up to 1,024 */
    size_t width;         /* the plan's, up to head_width */
    int layout;           /* FLINT_ROTARY_HALVES or FLINT_ROTARY_PAIRS */
    size_t q_stride;      /* values from a row to the next; multiples of 8 */
    size_t k_stride;
    size_t q_out_stride;
    size_t k_out_stride;
} flint_rotary_shape;

/* Rows of q (heads x head_width values, q_stride apart) turned by positions
 * (tokens int32 values of any sign, in device memory) into q_out, and k's into
 * k_out. q_out may be q itself with the same stride (in place), k_out k;
 * otherwise the outputs overlap neither each other nor an input. backward: by -t
 * instead (the gradients of q and k from those of q_out and k_out). A non-finite
 * value reaches its own pair, and no other value. */
FLINT_API flint_status flint_rotary(void* q_out, void* k_out, const void* q, const void* k,
                                    const void* positions, const void* plan,
                                    const flint_rotary_shape* shape, int backward,
                                    flint_stream stream);

#ifdef __cplusplus
}
#endif

#endif /* FLINT_FLINT_ROTARY_H */
