/*
 * hip_kv.h - C ABI of the MI355X (gfx950) rotary positions, the paged key and
 * value cache in 4 bits, and the attention that reads it.
 *
 * The chain between a step's q/k/v product and its output product, for
 * sequences of different lengths: hip_kv_append_dev rotates q and k and stores
 * k and v in 4 bits, hip_kv_attn_dev attends over the stored rows.
 * hip_lm_batch_new_kv4 (hip_lm.h) runs whole models on it.  The fp32
 * counterparts of the reference are rope_apply (nn.c:192-219), kvcache.c and
 * the attention of olmoe.c:214-341; it has no paged and no quantized cache.
 *
 * Conventions as hip_moe.h: plain C; 1 = done, 0 = not applicable or failed
 * (message in hip_moe_last_error()), and then nothing was enqueued; nothing
 * exits.  Every call enqueues on `stream` (a hipStream_t; NULL = the library's
 * stream for the current device) without waiting, and allocates, copies and
 * clears nothing: every call can be captured into a HIP graph.  Memory is
 * the caller's, on the current device.  Lengths, first rows and page tables
 * are read on the device, so a captured graph serves every step.
 *
 * Calls that read the same cache may overlap; a call that appends may overlap
 * with others only where they touch other pages.
 */
#ifndef HIP_KV_H
#define HIP_KV_H

#include <stddef.h>
#include <stdint.h>

#include "hip_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Types of q, k, v and outputs.  Sums and softmax statistics are fp32 for all of them.
 * What the attention multiplies is held in f16 parts: a query's value to 2^-22 of itself
 * (exactly in the 16-bit types) and 2^-38 (2^-34) of its head's largest, a probability
 * times its row's value scale to 2^-22 of itself (HIP_KV_BF16: 2^-11) and 2^-25 (16-bit
 * types: 2^-21) of the largest.  Whole outputs are 3e-7 to 5e-7 off in fp32, as far as
 * fp32 products and sums are, and by their own rounding in 16 bits.
 */
#define HIP_KV_F32 0
#define HIP_KV_F16 1
#define HIP_KV_BF16 2

/* ---------------------------------------------------------------------- */
/* rotary positions                                                       */
/* ---------------------------------------------------------------------- */

/* Which channels turn together: pair i is (2i, 2i + 1), as the reference's
 * rope_apply has them, or (i, i + rot / 2). */
#define HIP_ROPE_PAIRS 0
#define HIP_ROPE_HALVES 1

/* Frequencies stretched for contexts past the trained one (hip_rope_freqs). */
#define HIP_ROPE_PLAIN 0
#define HIP_ROPE_LINEAR 1 /* every frequency / factor */
#define HIP_ROPE_NTK 2    /* theta * factor^(rot / (rot - 2)) */
#define HIP_ROPE_YARN 3   /* by turns in the trained context: fast pairs keep theirs, slow ones / factor */

/*
 * A rotation: the first `rot` channels of a head (even, rot <= head length;
 * the others pass) turn by position * freq[i] radians, pair by pair:
 *   (a, b) -> mag * (a cos - b sin, b cos + a sin).
 * Angles, cosines and products are computed in 64 bits and rounded once.
 */
typedef struct hip_rope {
	size_t rot;
	int layout;         /* HIP_ROPE_PAIRS or HIP_ROPE_HALVES */
	const double *freq; /* device, [rot / 2] */
	double mag;         /* 1 for plain rotations */
} hip_rope;

/*
 * freq[rot / 2] and *mag on the host: freq[i] = theta^(-2i / rot), stretched
 * by `factor` (>= 1).  For HIP_ROPE_YARN, context is the trained length, and
 * pairs that turn more than fast times in it keep their frequency, those that
 * turn less than slow times take freq / factor, with a linear ramp over the
 * pairs between (0 for fast and slow: 32 and 1), and *mag = 0.1 ln(factor) + 1;
 * otherwise they are not read and *mag = 1.
 */
int hip_rope_freqs(size_t rot, double theta, int scaling, double factor, double context,
                   double fast, double slow, double *freq, double *mag);

/*
 * out = x rotated: rows of `heads` heads of head_len channels (1 .. 1024), row
 * r at x + r * x_stride elements, its position pos[r] (device, int32).  In
 * place where out == x and the strides are equal; otherwise x and out must not
 * overlap.
 */
int hip_rope_dev(const hip_rope *R, int type, const void *x, size_t x_stride, void *out,
                 size_t out_stride, size_t rows, size_t heads, size_t head_len,
                 const int32_t *pos, void *stream);

/* ---------------------------------------------------------------------- */
/* the cache                                                              */
/* ---------------------------------------------------------------------- */

/*
 * One layer's cache: `pages` pages of `page` rows (32, 64, .. 1024) each, for
 * kv_heads heads of head_len (64, 128 or 256) channels.  A page holds, head
 * after head, page / 32 tiles of 34 * head_len + 64 bytes, each 32 rows:
 *   key codes    uint32 [2][head_len / 32 / P][64][P], P = min(4, head_len / 32):
 *                word [t][a][16 * c + m][b] = row 16 t + m, channels
 *                32 (a P + b) + 8 c + (0 .. 7)
 *   value codes  uint32 [head_len / 64][64][4]: word [a][16 * c + m][b] =
 *                channel 64 a + 16 b + m, rows 4 c + (0 .. 3), 16 + 4 c + (0 .. 3)
 *   key scales   f16 [32][head_len / 32], one for 32 channels
 *   value scales f16 [32]
 * Code j (0 .. 7) of a word is in its bits 2 + 4 (j / 2) + 16 (j % 2) onwards
 * (the last two bits of code 7 wrap into bits 0 and 1).  A group of values
 * (32 channels of a key; a whole value row) is stored as Q4_0 does it: with m
 * its value of largest magnitude (the negative one of two equal), d = f16(m /
 * -8), held to +-65504, and code = floor(x / d + 8.5) within 0 .. 15; it stands
 * for d (code - 8).  Keys have a scale every 32 channels because their
 * channels differ most in size; a value row has one, which the attention
 * multiplies into the row's probability.  A group with a NaN has a NaN scale.
 * 138 bytes a row and head of 128 (fp32: 1024).
 */
typedef struct hip_kv_cache {
	void *pool; /* device, 16-byte aligned, pages * hip_kv_page_bytes */
	size_t pages, page, kv_heads, head_len;
	uint32_t *err; /* device word that HIP_KV_ERR_* bits are or'ed into, or NULL */
} hip_kv_cache;

#define HIP_KV_ERR_PAGE 1  /* a page id outside the pool: its rows were not stored, or not read */
#define HIP_KV_ERR_BATCH 2 /* a first row or length outside the batch's bounds: cut to them */

/* Bytes of one page; 0 if the shape is not one of the above. */
size_t hip_kv_page_bytes(size_t page, size_t kv_heads, size_t head_len);

/*
 * The rows of a call.  Sequence s has the rows row_start[s] .. row_start[s + 1]
 * - 1 of q, k, v and out, at the cache positions len[s] - n .. len[s] - 1 (n
 * its rows, len[s] its length with them).  Position p is row p % page of page
 * table[s * table_stride + p / page]; entries past the length, and in a windowed
 * call those before the window, may hold anything: they are not used, though an
 * attention without a window reads entries up to table_stride before it knows the
 * length.  A row at a position below 0 is not there: nothing is stored or read for
 * it, its place in a call's k, v and q_out is left as it was, and its attention is 0.
 */
typedef struct hip_kv_batch {
	size_t nseq;              /* 0 .. 65535; 0: nothing to do */
	size_t rows;              /* rows of all sequences, at most (below 2^31) */
	size_t max_rows;          /* rows of one sequence, at most */
	size_t max_len;           /* length of a sequence, at most (below 2^31 - 2^16) */
	const int32_t *row_start; /* device, [nseq + 1]; NULL: max_rows rows each */
	const int32_t *len;       /* device, [nseq] */
	const int32_t *table;     /* device, [nseq][table_stride] */
	size_t table_stride;      /* at least max_len / page, rounded up */
} hip_kv_batch;

/*
 * Store the batch's rows: k and v are rows of kv_heads * head_len values,
 * kv_stride elements apart.  With R, k turns first (its fp32 rounding is what
 * the codes are made of), by pos[row] (device) or, with pos NULL, by its
 * cache position.  With q (NULL: none), q_out = q rotated, rows of `heads`
 * heads; in place where q_out == q and the strides are equal.  Without R, q
 * must be NULL.  A call must not store into one page from two sequences, or from two
 * places of one.
 * Rows that are not the call's keep their bytes.  k, v, q and q_out are
 * 16-byte aligned, the strides multiples of 16 bytes.
 */
int hip_kv_append_dev(const hip_kv_cache *C, const hip_kv_batch *B, const hip_rope *R, int type,
                      const void *k, const void *v, size_t kv_stride, const int32_t *pos,
                      const void *q, size_t q_stride, size_t heads, void *q_out,
                      size_t q_out_stride, void *stream);

/*
 * The values that the batch's rows stand for, as k and v rows of kv_heads *
 * head_len values, `stride` elements apart (16-byte aligned, a multiple of
 * 16 bytes).  Rows that are not there, or on a page outside the pool, are
 * left as they were.
 */
int hip_kv_read_dev(const hip_kv_cache *C, const hip_kv_batch *B, int type, void *k, void *v,
                    size_t stride, void *stream);

/*
 * Causal attention of the batch's query rows, `heads` (a multiple of kv_heads;
 * head h reads kv head h / (heads / kv_heads)) heads of head_len: a row at
 * position p sees the cache positions p - window + 1 .. p (window 0: 0 .. p),
 *   out = sum_j softmax_j(scale q . k_j) v_j,
 * 0 for a row that is not there.  The scale is any finite number, the logits (scale
 * q . k_j) up to 2^21 in size, past which fp32 has no two of them nearer than 1/4.
 * q and out are 16-byte aligned with strides that are multiples of 16 bytes;
 * out == q with equal strides is allowed.
 * Rows outside the batch keep what out holds.  A row on a page outside the
 * pool is left out of the sum; where that leaves nothing the output is NaN.
 * ws: hip_kv_attn_ws bytes (of the same cache, bounds and heads, whatever the
 * window), 16-byte aligned, not used by another call at the same time (NULL if 0
 * bytes); graphs that may run at once need one each.  Where the heads of a kv head
 * times max_rows are 16 at most, a workspace serves every smaller max_len too.
 */
size_t hip_kv_attn_ws(const hip_kv_cache *C, const hip_kv_batch *B, size_t heads);
int hip_kv_attn_dev(const hip_kv_cache *C, const hip_kv_batch *B, int type, const void *q,
                    size_t q_stride, size_t heads, void *out, size_t out_stride, float scale,
                    size_t window, void *ws, size_t ws_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif
