/*
 * hip_f8.c - host layer of the 8-bit floating-point products
 * (include/hip_f8.h): the checks of the arguments, and the launches.  It keeps
 * no state.
 */
#include "hip_f8.h"
#include "f8_internal.h"
#include "moe_internal.h"

#include <hip/hip_runtime_api.h>
#include <stdarg.h>
#include <stdio.h>

static int f8_err(const char *fmt, ...)
{
	char buf[512];
	va_list ap;
	va_start(ap, fmt);
	vsnprintf(buf, sizeof(buf), fmt, ap);
	va_end(ap);
	moe_set_error(buf);
	return 0;
}

#define MAX_SIZE ((size_t)1 << 31)    /* strides: up to this; pairs: below it */
#define MAX_ROWS (MAX_SIZE - 65536)   /* rows and values of a row: below this, so that tiles that
					 end behind them are counted in 32 bits */
#define MAX_CODES ((size_t)1 << 24)   /* from row to row of codes: up to this, so that 256 rows'
					 distances fit 32 bits */
#define MAX_STRIDE ((size_t)1 << 40)  /* from matrix to matrix, of scales: up to this */
#define MAX_THREADS ((size_t)1 << 32) /* of one launch: below this */

static size_t type_bytes(int type)
{
	return type == HIP_F8_F32 ? 4 : 2;
}

static int check_type(const char *what, int type)
{
	if (type == HIP_F8_F32 || type == HIP_F8_F16 || type == HIP_F8_BF16)
		return 1;
	return f8_err("%s: unsupported type %d", what, type);
}

/* whether a launch of grid workgroups of `threads` can be made */
static int check_grid(const char *what, size_t a, size_t b, size_t threads)
{
	if (!a || !b || b <= (MAX_THREADS - 1) / threads / a)
		return 1;
	return f8_err("%s: too many rows and channels for one call", what);
}

/* rows of `width` values, `stride` apart, at p */
static int check_values(const char *what, const char *name, const void *p, size_t stride,
			size_t width, int type)
{
	if (!p)
		return f8_err("%s: NULL %s", what, name);
	if (stride < width || stride > MAX_SIZE)
		return f8_err("%s: %s rows of %zu values are %zu apart", what, name, width, stride);
	if ((uintptr_t)p % 16 || stride * type_bytes(type) % 16)
		return f8_err("%s: %s must be 16-byte aligned, its rows a multiple of 16 bytes apart",
			      what, name);
	return 1;
}

static int check_add(const char *what, const void *add, size_t add_stride, const void *out,
		     size_t out_stride, size_t n, int type)
{
	if (!add)
		return 1;
	if (add == out && add_stride != out_stride)
		return f8_err("%s: in place with two strides", what);
	return check_values(what, "add", add, add_stride ? add_stride : (n + 7) / 8 * 8, n, type);
}

static int check_rows(const char *what, const hip_f8_rows *X)
{
	if (X->k < 1 || X->k > F8_MAX_K)
		return f8_err("%s: rows of %zu channels (1 .. 2^20)", what, X->k);
	if (X->rows >= MAX_ROWS)
		return f8_err("%s: %zu rows (below 2^31 - 2^16)", what, X->rows);
	if (X->rows == 0)
		return 1;
	if (!X->codes || !X->scale)
		return f8_err("%s: NULL codes or scales of rows", what);
	if (X->stride < X->k || X->stride > MAX_CODES || X->stride % 16 || (uintptr_t)X->codes % 16)
		return f8_err("%s: rows of %zu codes are %zu apart (16-byte aligned, a multiple of 16 "
			      "up to 2^24)", what, X->k, X->stride);
	if (X->scale_stride < X->rows || X->scale_stride > MAX_SIZE || (uintptr_t)X->scale % 4)
		return f8_err("%s: scales of %zu rows are %zu apart (4-byte aligned)", what, X->rows,
			      X->scale_stride);
	return 1;
}

static int check_mat(const char *what, const char *name, const hip_f8_mat *W)
{
	if (W->n < 1 || W->n >= MAX_ROWS || W->k < 1 || W->k > F8_MAX_K)
		return f8_err("%s: %s of %zu rows of %zu columns (below 2^31 - 2^16 of 1 .. 2^20)", what, name,
			      W->n, W->k);
	if (W->count < 1 || W->count > F8_MAX_COUNT)
		return f8_err("%s: %zu matrices (1 .. 1024)", what, W->count);
	if (!W->codes || !W->scale)
		return f8_err("%s: NULL codes or scales of %s", what, name);
	if (W->stride < W->k || W->stride > MAX_CODES || W->stride % 16 || (uintptr_t)W->codes % 16)
		return f8_err("%s: %s rows of %zu codes are %zu apart (16-byte aligned, a multiple of 16 "
			      "up to 2^24)", what, name, W->k, W->stride);
	if (W->scale_stride < (W->k + HIP_F8_BLOCK - 1) / HIP_F8_BLOCK || W->scale_stride > MAX_SIZE ||
	    (uintptr_t)W->scale % 4)
		return f8_err("%s: %s scales of %zu columns are %zu apart (4-byte aligned)", what, name,
			      W->k, W->scale_stride);
	if (W->count > 1 && (W->step > MAX_STRIDE || W->scale_step > MAX_STRIDE || W->step % 16))
		return f8_err("%s: %s matrices %zu bytes and %zu scales apart (a multiple of 16, up to "
			      "2^40)", what, name, W->step, W->scale_step);
	return 1;
}

/* the stream of a call on the current device, which has to hold `mem`; 0 if
 * there is none */
static int call_stream(const char *what, const void *mem, void *stream, hipStream_t *s)
{
	int dev = 0, n = 0;
	if (hipGetDeviceCount(&n) != hipSuccess || n < 1 || hipGetDevice(&dev) != hipSuccess) {
		(void)hipGetLastError();
		return f8_err("%s: no HIP device", what);
	}
	if (n > 1 && mem) {
		hipPointerAttribute_t at;
		if (hipPointerGetAttributes(&at, mem) != hipSuccess) {
			(void)hipGetLastError();
			return f8_err("%s: memory that is not the device's", what);
		}
		if (at.device != dev)
			return f8_err("%s: memory of device %d, and device %d is current", what,
				      at.device, dev);
	}
	*s = stream ? (hipStream_t)stream : (hipStream_t)moe_device_stream(dev);
	return *s != NULL;
}

static int launched(const char *what, int rc)
{
	return rc == 0 ? 1 : f8_err("%s: %s", what, hipGetErrorString((hipError_t)rc));
}

int hip_f8_quantize_dev(int type, const void *x, size_t x_stride, const hip_f8_rows *X,
			void *stream)
{
	const char *what = "f8_quantize";
	hipStream_t s;
	if (!X)
		return f8_err("%s: NULL rows", what);
	if (!check_type(what, type) || !check_rows(what, X))
		return 0;
	if (X->rows == 0)
		return 1;
	if (!check_values(what, "x", x, x_stride, X->k, type) ||
	    !check_grid(what, f8_quantize_grid(X->rows, X->k), 1, F8_ROW_THREADS) ||
	    !call_stream(what, X->codes, stream, &s))
		return 0;
	return launched(what, f8_launch_quantize(type, x, x_stride, X, s));
}

/* a product's checks that the dense and the grouped form share, and its kernel form */
static int make_mul(const char *what, const hip_f8_rows *X, const hip_f8_mat *W,
		    const hip_f8_mat *up, int type, f8_mul_args *a)
{
	if (!X || !W)
		return f8_err("%s: NULL rows or matrix", what);
	if (!check_type(what, type) || !check_rows(what, X) || !check_mat(what, "matrix", W) ||
	    (up && !check_mat(what, "up", up)))
		return 0;
	if (X->k != W->k)
		return f8_err("%s: rows of %zu channels, matrices of %zu columns", what, X->k, W->k);
	if (up && (up->n != W->n || up->k != W->k || up->count != W->count))
		return f8_err("%s: %zu matrices of %zu x %zu, up of %zu of %zu x %zu", what, W->count,
			      W->n, W->k, up->count, up->n, up->k);
	const hip_f8_mat *m[2] = {W, up};
	for (int i = 0; i < 2; i++) {
		a->w[i] = m[i] ? m[i]->codes : NULL;
		a->ws[i] = m[i] ? m[i]->scale : NULL;
		a->w_stride[i] = m[i] ? (long)m[i]->stride : 0;
		a->ws_stride[i] = m[i] ? (long)m[i]->scale_stride : 0;
		a->w_step[i] = m[i] && m[i]->count > 1 ? (long)m[i]->step : 0;
		a->ws_step[i] = m[i] && m[i]->count > 1 ? (long)m[i]->scale_step : 0;
	}
	a->x = X->codes;
	a->xs = X->scale;
	a->x_stride = (long)X->stride;
	a->xs_stride = (long)X->scale_stride;
	a->x_rows = (int)X->rows;
	a->n = (int)W->n;
	a->k = (int)W->k;
	a->count = (int)W->count;
	return 1;
}

static int launch_mul(const char *what, f8_mul_args *a, int type, void *out, size_t out_stride,
		      void *stream)
{
	f8_plan p;
	hipStream_t s;
	if (!check_values(what, "out", out, out_stride, (size_t)a->n, type))
		return 0;
	a->out = out;
	a->out_stride = (long)out_stride;
	p.type = type;
	f8_mul_plan(a, &p);
	if (!check_grid(what, p.row_tiles, p.n_tiles, (size_t)p.threads) ||
	    !call_stream(what, out, stream, &s))
		return 0;
	return launched(what, f8_launch_mul(a, &p, s));
}

int hip_f8_mul_dev(const hip_f8_rows *X, const hip_f8_mat *W, const hip_f8_mat *up, int type,
		   const void *add, size_t add_stride, void *out, size_t out_stride,
		   void *stream)
{
	const char *what = "f8_mul";
	f8_mul_args a;
	if (!make_mul(what, X, W, up, type, &a))
		return 0;
	if (W->count != 1)
		return f8_err("%s: %zu matrices (1)", what, W->count);
	if (add && up)
		return f8_err("%s: an addend of a gated product", what);
	if (X->rows == 0)
		return 1;
	if (!check_add(what, add, add_stride, out, out_stride, W->n, type))
		return 0;
	a.from = a.start = NULL;
	a.add = add;
	a.add_stride = (long)add_stride;
	a.rows = a.x_rows;
	return launch_mul(what, &a, type, out, out_stride, stream);
}

int hip_f8_group_mul_dev(const hip_f8_rows *X, const int32_t *from, const int32_t *start,
			 size_t rows, const hip_f8_mat *W, const hip_f8_mat *up, int type,
			 void *out, size_t out_stride, void *stream)
{
	const char *what = "f8_group_mul";
	f8_mul_args a;
	if (!make_mul(what, X, W, up, type, &a))
		return 0;
	if (rows >= MAX_ROWS)
		return f8_err("%s: %zu rows (below 2^31 - 2^16)", what, rows);
	if (rows == 0)
		return 1;
	if (!start || (uintptr_t)start % 4 || (uintptr_t)from % 4)
		return f8_err("%s: NULL or misaligned rows of the experts", what);
	if (!from && X->rows < rows)
		return f8_err("%s: %zu rows of %zu", what, rows, X->rows);
	if (X->rows == 0)
		return f8_err("%s: %zu rows of none", what, rows);
	a.from = from;
	a.start = start;
	a.add = NULL;
	a.add_stride = 0;
	a.rows = (int)rows;
	return launch_mul(what, &a, type, out, out_stride, stream);
}

int hip_f8_sort_dev(const uint32_t *ids, size_t tokens, size_t topk, size_t experts,
		    int32_t *start, int32_t *from, int32_t *pos, void *stream)
{
	const char *what = "f8_sort";
	hipStream_t s;
	if (experts < 1 || experts > F8_MAX_COUNT)
		return f8_err("%s: %zu experts (1 .. 1024)", what, experts);
	if (topk < 1 || topk > F8_MAX_COUNT || tokens >= MAX_SIZE / topk)
		return f8_err("%s: %zu tokens of %zu slots (1 .. 1024; below 2^31 pairs)", what, tokens,
			      topk);
	if (!start || (tokens && (!ids || !from || !pos)))
		return f8_err("%s: NULL argument", what);
	if ((uintptr_t)ids % 4 || (uintptr_t)start % 4 || (uintptr_t)from % 4 || (uintptr_t)pos % 4)
		return f8_err("%s: misaligned pointer", what);
	if (!call_stream(what, start, stream, &s))
		return 0;
	return launched(what, f8_launch_sort(ids, (int)tokens, (int)topk, (int)experts, start, from, pos,
					     s));
}

int hip_f8_combine_dev(int type, const void *y, size_t y_stride, size_t y_rows,
		       const int32_t *pos, const float *w, size_t tokens, size_t topk, size_t n,
		       const void *add, size_t add_stride, void *out, size_t out_stride,
		       void *stream)
{
	const char *what = "f8_combine";
	hipStream_t s;
	if (!check_type(what, type))
		return 0;
	if (topk < 1 || topk > F8_MAX_COUNT || tokens >= MAX_SIZE / topk)
		return f8_err("%s: %zu tokens of %zu slots (1 .. 1024; below 2^31 pairs)", what, tokens,
			      topk);
	if (n < 1 || n >= MAX_ROWS || y_rows >= MAX_SIZE)
		return f8_err("%s: %zu rows of %zu values (below 2^31; 1 .. 2^31 - 2^16 - 1)", what, y_rows, n);
	if (tokens == 0)
		return 1;
	if (!pos || !w || (uintptr_t)pos % 4 || (uintptr_t)w % 4)
		return f8_err("%s: NULL or misaligned places or weights", what);
	if ((y_rows && !check_values(what, "y", y, y_stride, n, type)) ||
	    !check_values(what, "out", out, out_stride, n, type) ||
	    !check_add(what, add, add_stride, out, out_stride, n, type) ||
	    !check_grid(what, f8_combine_grid(type, tokens, n), 1, F8_ROW_THREADS) ||
	    !call_stream(what, out, stream, &s))
		return 0;
	return launched(what, f8_launch_combine(type, y, y_stride, (int)y_rows, pos, w, (int)tokens,
						(int)topk, (int)n, add, add_stride, out, out_stride, s));
}
