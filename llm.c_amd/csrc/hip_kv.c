/*
 * hip_kv.c - host layer of the rotary positions, the paged 4-bit cache and its
 * attention (include/hip_kv.h): the checks of the arguments, and the launches.
 * It keeps no state.
 */
#include "hip_kv.h"
#include "kv_internal.h"
#include "moe_internal.h"

#include <hip/hip_runtime_api.h>
#include <math.h>
#include <stdarg.h>
#include <stdio.h>

static int kv_err(const char *fmt, ...)
{
	char buf[512];
	va_list ap;
	va_start(ap, fmt);
	vsnprintf(buf, sizeof(buf), fmt, ap);
	va_end(ap);
	moe_set_error(buf);
	return 0;
}

#define MAX_GRID ((size_t)1 << 31) /* workgroups of one launch: below this */

/* workgroup count of the products of up to five factors, 0 past MAX_GRID */
static size_t grid_of(size_t a, size_t b, size_t c)
{
	if (!a || !b || !c)
		return 0;
	if (b > MAX_GRID / a || c > MAX_GRID / (a * b))
		return MAX_GRID;
	return a * b * c;
}

static size_t type_bytes(int type)
{
	return type == HIP_KV_F32 ? 4 : 2;
}

static int check_type(const char *what, int type)
{
	if (type == HIP_KV_F32 || type == HIP_KV_F16 || type == HIP_KV_BF16)
		return 1;
	return kv_err("%s: unsupported type %d", what, type);
}

static int check_rope(const char *what, const hip_rope *R, size_t head_len)
{
	if (!R->freq)
		return kv_err("%s: NULL frequencies", what);
	if (R->layout != HIP_ROPE_PAIRS && R->layout != HIP_ROPE_HALVES)
		return kv_err("%s: unknown layout %d", what, R->layout);
	if (R->rot < 2 || R->rot % 2 || R->rot > head_len)
		return kv_err("%s: %zu rotated channels of %zu (an even count from 2 on)", what, R->rot,
			      head_len);
	if ((uintptr_t)R->freq % 8)
		return kv_err("%s: misaligned frequencies", what);
	return 1;
}

/* rows of `width` values, `stride` apart, at p */
static int check_rows(const char *what, const char *name, const void *p, size_t stride,
		      size_t width, int type)
{
	if (!p)
		return kv_err("%s: NULL %s", what, name);
	if (stride < width)
		return kv_err("%s: %s rows of %zu values are %zu apart", what, name, width, stride);
	if (stride > (size_t)1 << 31)
		return kv_err("%s: %s rows are %zu values apart (2^31 at most)", what, name, stride);
	if ((uintptr_t)p % 16 || stride * type_bytes(type) % 16)
		return kv_err("%s: %s must be 16-byte aligned, its rows a multiple of 16 bytes apart",
			      what, name);
	return 1;
}

/* the stream of a call on the current device, which has to hold `mem` (NULL:
 * any); 0 if there is none */
static int call_stream(const char *what, const void *mem, void *stream, hipStream_t *s)
{
	int dev = 0, n = 0;
	if (hipGetDeviceCount(&n) != hipSuccess || n < 1 || hipGetDevice(&dev) != hipSuccess) {
		(void)hipGetLastError();
		return kv_err("%s: no HIP device", what);
	}
	if (n > 1 && mem) {
		hipPointerAttribute_t at;
		if (hipPointerGetAttributes(&at, mem) != hipSuccess) {
			(void)hipGetLastError();
			return kv_err("%s: memory that is not the device's", what);
		}
		if (at.device != dev)
			return kv_err("%s: memory of device %d, and device %d is current", what,
				      at.device, dev);
	}
	*s = stream ? (hipStream_t)stream : (hipStream_t)moe_device_stream(dev);
	return *s != NULL;
}

static int launched(const char *what, int rc)
{
	return rc == 0 ? 1 : kv_err("%s: %s", what, hipGetErrorString((hipError_t)rc));
}

int hip_rope_freqs(size_t rot, double theta, int scaling, double factor, double context,
		   double fast, double slow, double *freq, double *mag)
{
	if (!freq || !mag)
		return kv_err("rope_freqs: NULL argument");
	if (rot < 2 || rot % 2 || rot > 1024)
		return kv_err("rope_freqs: %zu rotated channels (an even count, 2 .. 1024)", rot);
	if (!(theta > 1.0) || !isfinite(theta))
		return kv_err("rope_freqs: theta %g (above 1)", theta);
	if (scaling < HIP_ROPE_PLAIN || scaling > HIP_ROPE_YARN)
		return kv_err("rope_freqs: unknown scaling %d", scaling);
	if (scaling != HIP_ROPE_PLAIN && (!(factor >= 1.0) || !isfinite(factor)))
		return kv_err("rope_freqs: factor %g (1 or more)", factor);
	fast = fast == 0.0 ? 32.0 : fast;
	slow = slow == 0.0 ? 1.0 : slow;
	if (scaling == HIP_ROPE_YARN &&
	    (!(context > 0.0) || !isfinite(context) || !(slow > 0.0) || !(fast >= slow) || !isfinite(fast)))
		return kv_err("rope_freqs: context %g, turns %g and %g", context, fast, slow);
	if (scaling == HIP_ROPE_NTK && rot > 2)
		theta *= pow(factor, (double)rot / (double)(rot - 2));
	/* the pair that turns n times in the context: rot * ln(context / 2 pi n) /
	 * (2 ln theta) */
	double lo = 0.0, hi = 0.0;
	*mag = 1.0;
	if (scaling == HIP_ROPE_YARN) {
		const double tau = 6.283185307179586476925;
		lo = floor((double)rot * log(context / (fast * tau)) / (2.0 * log(theta)));
		hi = ceil((double)rot * log(context / (slow * tau)) / (2.0 * log(theta)));
		lo = lo > 0.0 ? lo : 0.0;
		hi = hi < (double)rot - 1.0 ? hi : (double)rot - 1.0;
		*mag = 0.1 * log(factor) + 1.0;
	}
	const double width = hi - lo > 1e-3 ? hi - lo : 1e-3;
	for (size_t i = 0; i < rot / 2; i++) {
		double f = pow(theta, -2.0 * (double)i / (double)rot);
		if (scaling == HIP_ROPE_LINEAR)
			f /= factor;
		if (scaling == HIP_ROPE_YARN) {
			double ramp = ((double)i - lo) / width;
			ramp = ramp < 0.0 ? 0.0 : ramp > 1.0 ? 1.0 : ramp;
			f = f / factor * ramp + f * (1.0 - ramp);
		}
		freq[i] = f;
	}
	return 1;
}

int hip_rope_dev(const hip_rope *R, int type, const void *x, size_t x_stride, void *out,
		 size_t out_stride, size_t rows, size_t heads, size_t head_len,
		 const int32_t *pos, void *stream)
{
	const char *what = "rope";
	hipStream_t s;
	if (!R || !x || !out || !pos)
		return kv_err("%s: NULL argument", what);
	if (head_len < 1 || head_len > 1024 || heads < 1 || heads > 65536)
		return kv_err("%s: %zu heads of %zu channels (1 .. 65536 of 1 .. 1024)", what, heads,
			      head_len);
	if (!check_type(what, type) || !check_rope(what, R, head_len))
		return 0;
	if (rows >= (size_t)1 << 31)
		return kv_err("%s: %zu rows (below 2^31)", what, rows);
	if (x_stride < heads * head_len || out_stride < heads * head_len || x_stride > (size_t)1 << 31 ||
	    out_stride > (size_t)1 << 31)
		return kv_err("%s: rows of %zu values are %zu and %zu apart", what, heads * head_len,
			      x_stride, out_stride);
	if ((uintptr_t)x % type_bytes(type) || (uintptr_t)out % type_bytes(type) || (uintptr_t)pos % 4)
		return kv_err("%s: misaligned pointer", what);
	if (x == out && x_stride != out_stride)
		return kv_err("%s: in place with two strides", what);
	if (rows == 0)
		return 1;
	if (!call_stream(what, x, stream, &s))
		return 0;
	return launched(what, kv_launch_rope(type, x, x_stride, out, out_stride, rows, (int)heads,
					     (int)head_len, R, pos, s));
}

size_t hip_kv_page_bytes(size_t page, size_t kv_heads, size_t head_len)
{
	if (page < KV_TILE || page > 1024 || (page & (page - 1)) || kv_heads < 1 || kv_heads > 4096 ||
	    (head_len != 64 && head_len != 128 && head_len != 256))
		return 0;
	return page / KV_TILE * kv_heads * (34 * head_len + 64);
}

/* the checks of a cache and a batch, and their kernel form; 2: no rows */
static int make_args(const char *what, const hip_kv_cache *C, const hip_kv_batch *B, kv_args *a)
{
	if (!C || !B)
		return kv_err("%s: NULL cache or batch", what);
	if (!hip_kv_page_bytes(C->page, C->kv_heads, C->head_len))
		return kv_err("%s: pages of %zu rows of %zu heads of %zu channels (32, 64 .. 1024 rows, 1 .. "
			      "4096 heads of 64, 128 or 256)", what, C->page, C->kv_heads, C->head_len);
	if (C->pages >= (size_t)1 << 31)
		return kv_err("%s: %zu pages (below 2^31)", what, C->pages);
	if (B->nseq > 65535)
		return kv_err("%s: %zu sequences (65535 at most)", what, B->nseq);
	if (B->rows >= (size_t)1 << 31 || B->max_rows > B->rows)
		return kv_err("%s: %zu rows, %zu of one sequence", what, B->rows, B->max_rows);
	if (B->max_len >= ((size_t)1 << 31) - ((size_t)1 << 16))
		return kv_err("%s: sequences of %zu rows (below 2^31 - 2^16)", what, B->max_len);
	if (B->nseq == 0 || B->max_rows == 0)
		return 2;
	if (!B->row_start && B->max_rows > B->rows / B->nseq)
		return kv_err("%s: %zu sequences of %zu rows are more than %zu", what, B->nseq,
			      B->max_rows, B->rows);
	if (!C->pool || !B->len || !B->table)
		return kv_err("%s: NULL pool, lengths or page table", what);
	if ((uintptr_t)C->pool % 16 || (uintptr_t)C->err % 4 || (uintptr_t)B->row_start % 4 ||
	    (uintptr_t)B->len % 4 || (uintptr_t)B->table % 4)
		return kv_err("%s: misaligned pool (16 bytes), lengths or page table", what);
	if (B->table_stride < (B->max_len + C->page - 1) / C->page || B->table_stride >= (size_t)1 << 31)
		return kv_err("%s: page tables of %zu entries for %zu rows in pages of %zu", what,
			      B->table_stride, B->max_len, C->page);
	a->pool = C->pool;
	a->err = C->err;
	a->row_start = B->row_start;
	a->len = B->len;
	a->table = B->table;
	a->table_stride = (long)B->table_stride;
	a->pages = (int)C->pages;
	a->page_shift = __builtin_ctz((unsigned)C->page);
	a->kv_heads = (int)C->kv_heads;
	a->nseq = (int)B->nseq;
	a->rows = (int)B->rows;
	a->max_rows = (int)B->max_rows;
	a->max_len = (int)B->max_len;
	if (grid_of(B->nseq, 4 * (B->max_rows / KV_TILE + 2), C->kv_heads) >= MAX_GRID)
		return kv_err("%s: %zu sequences of up to %zu rows are too many for one call", what,
			      B->nseq, B->max_rows);
	return 1;
}

int hip_kv_append_dev(const hip_kv_cache *C, const hip_kv_batch *B, const hip_rope *R, int type,
		      const void *k, const void *v, size_t kv_stride, const int32_t *pos,
		      const void *q, size_t q_stride, size_t heads, void *q_out,
		      size_t q_out_stride, void *stream)
{
	const char *what = "kv_append";
	kv_args a;
	hipStream_t s;
	const int ok = make_args(what, C, B, &a);
	if (!ok || !check_type(what, type) || (R && !check_rope(what, R, C->head_len)))
		return 0;
	const size_t width = C->kv_heads * C->head_len;
	if (q && !R)
		return kv_err("%s: queries without a rotation", what);
	if (q && (heads < 1 || heads > 65536))
		return kv_err("%s: %zu query heads (1 .. 65536)", what, heads);
	if (ok == 2)
		return 1;
	if (!check_rows(what, "k", k, kv_stride, width, type) ||
	    !check_rows(what, "v", v, kv_stride, width, type) ||
	    (q && (!check_rows(what, "q", q, q_stride, heads * C->head_len, type) ||
		   !check_rows(what, "q_out", q_out, q_out_stride, heads * C->head_len, type))))
		return 0;
	if (q && q == q_out && q_stride != q_out_stride)
		return kv_err("%s: queries in place with two strides", what);
	if ((uintptr_t)pos % 4)
		return kv_err("%s: misaligned positions", what);
	if (!call_stream(what, C->pool, stream, &s))
		return 0;
	return launched(what, kv_launch_append(&a, (int)C->head_len, type, R, k, v, kv_stride, pos, q,
					       q_stride, (int)heads, q_out, q_out_stride, s));
}

int hip_kv_read_dev(const hip_kv_cache *C, const hip_kv_batch *B, int type, void *k, void *v,
		    size_t stride, void *stream)
{
	const char *what = "kv_read";
	kv_args a;
	hipStream_t s;
	const int ok = make_args(what, C, B, &a);
	if (!ok || !check_type(what, type))
		return 0;
	if (ok == 2)
		return 1;
	if (!check_rows(what, "k", k, stride, C->kv_heads * C->head_len, type) ||
	    !check_rows(what, "v", v, stride, C->kv_heads * C->head_len, type))
		return 0;
	if (!call_stream(what, C->pool, stream, &s))
		return 0;
	return launched(what, kv_launch_read(&a, (int)C->head_len, type, k, v, stride, s));
}

/* the attention's plan; 2: no rows */
static int attn_plan(const char *what, const hip_kv_cache *C, const hip_kv_batch *B, size_t heads,
		     size_t window, kv_args *a, kv_plan *p, int *w)
{
	const int ok = make_args(what, C, B, a);
	if (!ok)
		return 0;
	if (heads < 1 || heads > 65536 || heads % C->kv_heads)
		return kv_err("%s: %zu query heads on %zu kv heads", what, heads, C->kv_heads);
	if (ok == 2)
		return 2;
	if (B->max_rows > ((size_t)1 << 30) / (heads / C->kv_heads))
		return kv_err("%s: %zu rows of one sequence are too many for one call", what,
			      B->max_rows);
	*w = window >= B->max_len ? 0 : (int)window;
	kv_attn_plan(a, (int)C->head_len, (int)heads, *w, p);
	if (grid_of(grid_of(B->nseq, C->kv_heads, (size_t)p->row_tiles), (size_t)p->splits, 1) >= MAX_GRID)
		return kv_err("%s: %zu sequences of up to %zu rows are too many for one call", what,
			      B->nseq, B->max_rows);
	return 1;
}

size_t hip_kv_attn_ws(const hip_kv_cache *C, const hip_kv_batch *B, size_t heads)
{
	kv_args a;
	kv_plan p;
	int w;
	return attn_plan("kv_attn_ws", C, B, heads, 0, &a, &p, &w) == 1 ? p.ws : 0;
}

int hip_kv_attn_dev(const hip_kv_cache *C, const hip_kv_batch *B, int type, const void *q,
		    size_t q_stride, size_t heads, void *out, size_t out_stride, float scale,
		    size_t window, void *ws, size_t ws_bytes, void *stream)
{
	const char *what = "kv_attn";
	kv_args a;
	kv_plan p;
	hipStream_t s;
	int w = 0;
	const int ok = attn_plan(what, C, B, heads, window, &a, &p, &w);
	if (!ok || !check_type(what, type))
		return 0;
	if (!isfinite(scale))
		return kv_err("%s: scale %g", what, (double)scale);
	if (ok == 2)
		return 1;
	if (!check_rows(what, "q", q, q_stride, heads * C->head_len, type) ||
	    !check_rows(what, "out", out, out_stride, heads * C->head_len, type))
		return 0;
	if (q == out && q_stride != out_stride)
		return kv_err("%s: in place with two strides", what);
	if (p.ws && (!ws || (uintptr_t)ws % 16 || ws_bytes < p.ws))
		return kv_err("%s: a workspace of %zu bytes at %p, %zu are needed (16-byte aligned)", what,
			      ws_bytes, ws, p.ws);
	if (!call_stream(what, C->pool, stream, &s))
		return 0;
	return launched(what, kv_launch_attn(&a, (int)C->head_len, type, q, q_stride, (int)heads, out,
					     out_stride, scale, w, ws, &p, s));
}
