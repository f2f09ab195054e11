/*
 * Internal interface between the host layer (hip_kv.c) and the kernels of the
 * rotary positions and the 4-bit cache (kv_cache.hip, kv_attn.hip).  Launchers
 * return a hipError_t value (0 = success) and enqueue on the given stream
 * without waiting; the host has checked every argument.
 */
#ifndef KV_INTERNAL_H
#define KV_INTERNAL_H

#include <stddef.h>
#include <stdint.h>

#include "hip_kv.h"

#ifdef __cplusplus
extern "C" {
#endif

#define KV_TILE 32 /* cached rows of one tile */
#define KV_MAX_HEAD_LEN 256

/* a cache and a batch as the kernels take them */
typedef struct kv_args {
	uint8_t *pool;
	uint32_t *err;
	const int32_t *row_start, *len, *table;
	long table_stride;
	int pages, page_shift, kv_heads, nseq, rows, max_rows, max_len;
} kv_args;

int kv_launch_rope(int type, const void *x, size_t x_stride, void *out, size_t out_stride,
                   size_t rows, int heads, int head_len, const hip_rope *R, const int32_t *pos,
                   void *stream);
int kv_launch_append(const kv_args *a, int head_len, int type, const hip_rope *R, const void *k,
                     const void *v, size_t kv_stride, const int32_t *pos, const void *q,
                     size_t q_stride, int heads, void *q_out, size_t q_out_stride, void *stream);
int kv_launch_read(const kv_args *a, int head_len, int type, void *k, void *v, size_t stride,
                   void *stream);

/* how an attention call is cut up, from the host's bounds alone */
typedef struct kv_plan {
	int row_tiles; /* tiles of query rows of one (sequence, kv head) */
	int wide;      /* tiles of 32 query rows */
	int rows;      /* query rows of a tile, at most */
	int slots;     /* columns of a query row */
	int waves;     /* of a workgroup */
	int chunk;     /* cache tiles of one workgroup */
	int splits;    /* workgroups along the cache */
	int shares;    /* of all caches together, for each kv head, instead (0: no) */
	size_t ws;     /* bytes of partial results, whatever the window */
} kv_plan;
void kv_attn_plan(const kv_args *a, int head_len, int heads, int window, kv_plan *p);
int kv_launch_attn(const kv_args *a, int head_len, int type, const void *q, size_t q_stride,
                   int heads, void *out, size_t out_stride, float scale, int window, void *ws,
                   const kv_plan *p, void *stream);

#ifdef __cplusplus
}
#endif
#endif
