/*
 * Internal interface between the host layer (hip_f8.c) and the kernels of the
 * 8-bit floating-point products (f8_rows.hip, f8_mul.hip).  Launchers return a
 * hipError_t value (0 = success) and enqueue on the given stream without waiting;
 * the host has checked every argument.
 */
#ifndef F8_INTERNAL_H
#define F8_INTERNAL_H

#include <stddef.h>
#include <stdint.h>

#include "hip_f8.h"

#ifdef __cplusplus
extern "C" {
#endif

#define F8_MAX_COUNT 1024 /* experts of one call */
#define F8_MAX_K ((size_t)1 << 20)

/* a product as the kernels take it: W and, gated, up */
typedef struct f8_mul_args {
	const uint8_t *x;
	const float *xs;
	const uint8_t *w[2];
	const float *ws[2];
	const int32_t *from, *start; /* NULL: rows as they come; one matrix for all */
	const void *add;
	void *out;
	long x_stride, xs_stride, w_stride[2], ws_stride[2], w_step[2], ws_step[2];
	long add_stride, out_stride;
	int x_rows, rows, n, k, count;
} f8_mul_args;

/* how a product is cut up, from the host's bounds alone */
typedef struct f8_plan {
	int type;         /* set by the caller */
	int form;         /* of f8_mul.hip's */
	size_t row_tiles; /* tiles of rows, at most, over all experts */
	size_t n_tiles;
	int threads;
} f8_plan;
void f8_mul_plan(const f8_mul_args *a, f8_plan *p);
int f8_launch_mul(const f8_mul_args *a, const f8_plan *p, void *stream);

size_t f8_quantize_grid(size_t rows, size_t k);
int f8_launch_quantize(int type, const void *x, size_t x_stride, const hip_f8_rows *X, void *stream);
int f8_launch_sort(const uint32_t *ids, int tokens, int topk, int experts, int32_t *start,
                   int32_t *from, int32_t *pos, void *stream);
size_t f8_combine_grid(int type, size_t tokens, size_t n);
int f8_launch_combine(int type, const void *y, size_t y_stride, int y_rows, const int32_t *pos,
                      const float *w, int tokens, int topk, int n, const void *add,
                      size_t add_stride, void *out, size_t out_stride, void *stream);
#define F8_ROW_THREADS 256 /* of the quantizer's and the combine's workgroups */

#ifdef __cplusplus
}
#endif
#endif
