/*
 * hip_f8.h - C ABI of the MI355X (gfx950) products in 8-bit floating point:
 * weights as e4m3 codes with a scale for each block of 128 x 128, rows as e4m3
 * codes with a scale for each 128 channels.
 *
 * The experts' part of a mixture-of-experts layer whose weights come in this form
 * instead of GGUF blocks, from the ids and weights that hip_moe_route_dev gives:
 *   hip_f8_sort_dev      the (token, slot) pairs by expert
 *   hip_f8_quantize_dev  the tokens
 *   hip_f8_group_mul_dev silu(gate) * up of every expert's rows
 *   hip_f8_quantize_dev  those
 *   hip_f8_group_mul_dev down
 *   hip_f8_combine_dev   the weighted sum per token
 * and the dense product (hip_f8_mul_dev), next to hip_moe_qmat_mul_dev.  The
 * reference's counterparts, in its own formats, are moe_ffn (olmoe.c:343-407) and
 * tensor_mma_transposed_2x2 (matmul.c:451-462); it has no 8-bit floating point.
 *
 * Conventions as hip_moe.h: plain C; 1 = done, 0 = not applicable or failed
 * (message in hip_moe_last_error()), and then nothing was enqueued; nothing
 * exits.  Every call enqueues on `stream` (a hipStream_t; NULL = the library's
 * stream for the current device) without waiting, and allocates, copies and
 * clears nothing: every call can be captured into a HIP graph, needs no
 * workspace, and calls may overlap where none writes what another reads or
 * writes.  Memory is the caller's, on the current device.  Inputs and outputs
 * do not overlap unless a call says so.  Of a row of inputs that ends inside 16
 * bytes, counted from its start, the rest of them may be read too (they are aligned
 * and in the same page); what is there does not matter.  A call whose launch would have
 * 2^32 threads or more is refused.  Results do not depend on timing: the same call
 * gives the same bits.
 */
#ifndef HIP_F8_H
#define HIP_F8_H

#include <stddef.h>
#include <stdint.h>

#include "hip_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Types of inputs and outputs that are not codes. */
#define HIP_F8_F32 0
#define HIP_F8_F16 1
#define HIP_F8_BF16 2

/* Channels (and, in a matrix, rows) that share a scale. */
#define HIP_F8_BLOCK 128

/*
 * Codes are e4m3: sign, 4 bits of exponent (bias 7), 3 of mantissa; 0x7f and 0xff
 * are NaN, there are no infinities, the largest value is 448, the smallest 2^-9.
 *
 * Quantized rows.  Channel c of row r stands for
 *   e4m3(codes[r * stride + c]) * scale[c / 128 * scale_stride + r],
 * so that the scales of neighbouring rows lie next to each other.  The codes are
 * 16-byte aligned, the stride a multiple of 16, at least k and at most 2^24; bytes between k and
 * the stride may hold anything.
 */
typedef struct hip_f8_rows {
	uint8_t *codes; /* device, rows * stride bytes */
	size_t stride;
	float *scale; /* device, [(k + 127) / 128][scale_stride] */
	size_t scale_stride; /* at least rows */
	size_t rows, k; /* below 2^31 - 2^16; 1 .. 2^20 */
} hip_f8_rows;

/*
 * `count` matrices of n rows of k columns.  Column c of row r of matrix e stands for
 *   e4m3(codes[e * step + r * stride + c]) *
 *   scale[e * scale_step + r / 128 * scale_stride + c / 128].
 * The codes are 16-byte aligned, stride and step multiples of 16, the stride at most
 * 2^24; bytes between k and the stride may hold anything.
 */
typedef struct hip_f8_mat {
	const uint8_t *codes; /* device */
	size_t stride;        /* bytes from row to row, at least k */
	const float *scale;   /* device */
	size_t scale_stride;  /* at least (k + 127) / 128 */
	size_t n, k;          /* 1 .. 2^31 - 2^16 - 1, 1 .. 2^20 */
	size_t count;         /* 1 .. 1024 */
	size_t step, scale_step; /* from matrix to matrix; not read where count is 1 */
} hip_f8_mat;

/*
 * Quantize rows: X->rows rows of X->k values, x_stride values apart, 16-byte
 * aligned with rows a multiple of 16 bytes apart.  For each 128 channels (the last
 * may be fewer) with largest magnitude m:
 *   scale = max(fl(m / 448), 2^-96),  code = the e4m3 value nearest to x / scale,
 * ties to even, the quotient not rounded before.  A block that holds a NaN or an
 * infinity has a NaN scale and codes of 0.  Bytes of X's rows from k to the next
 * multiple of 16 become 0.
 */
int hip_f8_quantize_dev(int type, const void *x, size_t x_stride, const hip_f8_rows *X,
                        void *stream);

/*
 * out = X W^T (+ add), or with `up` (of W's n, k and count; else NULL)
 * out = silu(X W^T) * (X up^T), silu(a) = a / (1 + exp(-a)), for which 0 may stand where
 * it is smaller than 2^-119: X->rows rows of W->n values, out_stride values apart; W->count
 * is 1.  add: rows of the same type, add_stride values apart, or one row for all
 * (add_stride 0), or NULL; with `up` it is NULL.  add == out is allowed with equal strides.
 * out and add are 16-byte aligned, rows a multiple of 16 bytes apart.
 * A block's products are summed up and join the others' sum times the product of both
 * scales, in fp32; one rounding to the type at the end.  For fp32 outputs the products
 * are exact and the sums fp32's: off by (2^-17 + (k / 128 + 3) 2^-24) sum |x w| at most,
 * whole outputs by 1e-7 at 4096 channels.  For 16-bit outputs the matrix cores cut each of
 * eight products that they add up at 2^-13 of the largest one's power of two: off by 2^-10
 * sum |x w| more at most, whole outputs by 1.3e-5 to 3e-5 (channels of very different size),
 * and by that rounding (1.7e-3 bf16, 2.1e-4 f16).  The product of two scales is rounded to
 * fp32: where it is below 2^-126 to a multiple of 2^-149, which is that much more, and where
 * it is no finite number, outputs may be NaN.
 */
int hip_f8_mul_dev(const hip_f8_rows *X, const hip_f8_mat *W, const hip_f8_mat *up, int type,
                   const void *add, size_t add_stride, void *out, size_t out_stride,
                   void *stream);

/*
 * Pairs by expert.  ids[tokens][topk] (device); pair t * topk + s has expert
 * ids[t * topk + s], or none of this call's if that is `experts` (1 .. 1024) or more.
 * Pairs of one expert keep their order:
 *   start[e] .. start[e + 1] - 1   the rows of expert e ([experts + 1])
 *   from[row]                      the row's token ([tokens * topk]; from start[experts] on
 *                                  left as it was)
 *   pos[t * topk + s]              the pair's row, -1 if it has none
 * tokens * topk is below 2^31.
 */
int hip_f8_sort_dev(const uint32_t *ids, size_t tokens, size_t topk, size_t experts,
                    int32_t *start, int32_t *from, int32_t *pos, void *stream);

/*
 * The product of each expert's rows with its matrix: out row r of start[e] <= r <
 * start[e + 1] (device, [W->count + 1], not decreasing) is row from[r] of X, or with
 * from NULL row r of X, times matrix e; with `up` gated as above.  `rows`: the rows
 * of out, at least start[W->count]; others keep what out holds.  A row whose from is
 * outside X's rows is NaN.
 */
int hip_f8_group_mul_dev(const hip_f8_rows *X, const int32_t *from, const int32_t *start,
                         size_t rows, const hip_f8_mat *W, const hip_f8_mat *up, int type,
                         void *out, size_t out_stride, void *stream);

/*
 * out[t] = add[t] + sum_s w[t * topk + s] * y[pos[t * topk + s]], slot after slot in fp32,
 * over the slots whose pos is a row of y (0 .. y_rows - 1): rows of n values, y_stride,
 * add_stride and out_stride values apart, all of one type, 16-byte aligned, rows a
 * multiple of 16 bytes apart; add as above.  A weight whose slot has no row is not read.
 */
int hip_f8_combine_dev(int type, const void *y, size_t y_stride, size_t y_rows,
                       const int32_t *pos, const float *w, size_t tokens, size_t topk, size_t n,
                       const void *add, size_t add_stride, void *out, size_t out_stride,
                       void *stream);

#ifdef __cplusplus
}
#endif
#endif
