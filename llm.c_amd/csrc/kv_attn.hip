/*
 * kv_attn.hip - causal attention of query rows over the paged 4-bit cache
 * (include/hip_kv.h), on the gfx950 matrix cores.
 *
 * The rows of one (sequence, kv head) are its query rows times the query heads
 * that share the kv head, row by row (row i, head g: i * G + g), in tiles of
 * 16.  A wave takes one such tile over 32 cached rows at a time, everything
 * with the query rows in the MFMA's columns:
 *   S^T [cached row][query row] = K . Q^T     v_mfma_f32_16x16x32_f16, a step
 *                                             for each 32-channel group
 *   O^T [channel][query row] += V^T . P^T     the same, a step for each 16 channels
 * so a lane holds one query row (lane % 16) throughout: its softmax maximum
 * and sum are one register each, the rescaling of O needs no exchange, and the
 * scores come out of the first product in the lanes in which the second takes
 * the probabilities (the cached rows of a lane, 4 c .. 4 c + 3 of each half of
 * the tile, c = lane / 16, are the eight that a value word holds).
 *
 * Exactness.  Codes are small integers, exact in f16, and stay unscaled in the
 * operands: a key group's scale multiplies its partial scores in fp32, a value
 * row's scale its probability.  A key code q enters as the subnormal q * 2^-18
 * (its bits in place, nothing around them) and its surplus of 8 a channel leaves
 * through the accumulator's start (-8 sum of the query's channels); a value code
 * enters as 16 + q (its bits or'ed into the mantissa of 16.0) less 24, since over
 * many cached rows a surplus would outweigh the sum.  A query row is scaled by a power of two (its largest value into [2^13, 2^14))
 * and, from fp32, split into two f16 parts of together 22 bits; f16 and bf16
 * queries are exact in one.  The probability times the value scale is scaled
 * by a power of two that keeps the largest below 2^15, and split in two as
 * well (in one part, 11 bits, for bf16 outputs of 8).  Sums, maxima and
 * exponents are fp32.
 */
#include "kv_device.h"

#define KV_NT 256
#define KV_WAVES (KV_NT / WAVE)
#define KV_ROWS 16 /* query rows of a tile */

__device__ static inline half8_t as_half8(u32 a, u32 b, u32 c, u32 d)
{
	const u32x4 v = {a, b, c, d};
	return __builtin_bit_cast(half8_t, v);
}

/* a word's codes, in their order, as f16 with the mantissa's upper four bits:
 * code * 2^-18, or with base = 0x4c004c00 16 + code */
__device__ static inline half8_t kv_word(u32 w, u32 base)
{
	const u32 m = 0x03c003c0u; /* the codes whose lowest bits are 6 and 22 */
	return as_half8((w << 4 & m) | base, (w & m) | base, (w >> 4 & m) | base,
			(kv_rotr(w, 8) & m) | base);
}

#define KV_CODE_STEP (1.0f / (1 << 18))

/* the largest over the four lanes that share a query row */
__device__ static inline float row_max(float v)
{
	v = fmaxf(v, __shfl_xor(v, 16, WAVE));
	return fmaxf(v, __shfl_xor(v, 32, WAVE));
}

__device__ static inline float row_sum(float v)
{
	v += __shfl_xor(v, 16, WAVE);
	return v + __shfl_xor(v, 32, WAVE);
}

/* 2^n, n within -126 .. 127 */
__device__ static inline float pow2(int n)
{
	return __builtin_bit_cast(float, (u32)(n + 127) << 23);
}

/* the exponent e of v = m 2^e, 0.5 <= m < 1 (finite, not 0) */
__device__ static inline int exponent(float v)
{
	return __builtin_amdgcn_frexp_expf(v);
}

/* the rows that a tile of query rows sees: the lane's row, and all of them */
struct kv_span {
	int lo, hi;         /* cached rows of the lane's query row */
	int first, last;    /* of all rows of the tile */
	int inner0, inner1; /* seen by every row of the tile */
	size_t at;          /* the row's index among the batch's rows, and its head */
	int head;
	bool valid;
};

__device__ static inline kv_span kv_rows_of(const kv_seq &sq, int tile, int G, int kv_head, int window,
					    int lane)
{
	kv_span r;
	const int base = sq.len - sq.n, all = sq.n * G;
	const int mine = tile * KV_ROWS + lane % 16;
	const int i0 = tile * KV_ROWS / G, i1 = (min(tile * KV_ROWS + KV_ROWS, all) - 1) / G;
	const int i = min(mine, all - 1) / G;
	r.valid = mine < all;
	r.hi = base + i + 1;
	r.lo = window ? max(0, r.hi - window) : 0;
	r.at = sq.row + i;
	r.head = kv_head * G + min(mine, all - 1) % G;
	r.last = base + i1 + 1;
	r.first = window ? max(0, base + i0 + 1 - window) : 0;
	r.inner0 = window ? max(0, r.last - window) : 0;
	r.inner1 = base + i0 + 1;
	return r;
}

/*
 * One workgroup: a tile of query rows over `chunk` tiles of the cache, dealt to
 * its four waves one by one; the waves' results meet in LDS.  With more than
 * one workgroup along the cache each leaves its maximum, sum and unnormalised
 * output in ws for k_kv_merge.
 */
template <int D, int TY>
__global__ __launch_bounds__(KV_NT) void k_kv_attn(
	kv_args a, const typename kv_type<TY>::t *q, size_t q_stride, int G,
	typename kv_type<TY>::t *out, size_t out_stride, float scale, int window, float *ws,
	int row_tiles, int chunk, int splits)
{
	typedef kv_type<TY> T;
	typedef kv_tile<D> L;
	constexpr int QP = TY == HIP_KV_F32 ? 2 : 1, PP = TY == HIP_KV_BF16 ? 1 : 2;
	constexpr int CT = D / 16; /* channel tiles of O^T */
	__shared__ float s_o[KV_WAVES][KV_ROWS][D + 4];
	__shared__ float s_m[KV_WAVES][KV_ROWS], s_l[KV_WAVES][KV_ROWS];

	const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE, part = lane / 16;
	int b = blockIdx.x;
	const int kv_head = b % a.kv_heads;
	b /= a.kv_heads;
	const int split = b % splits;
	b /= splits;
	const int rt = b % row_tiles, s = b / row_tiles;
	const kv_seq sq = kv_sequence(a, s);
	if (rt * KV_ROWS >= sq.n * G)
		return;
	const kv_span r = kv_rows_of(sq, rt, G, kv_head, window, lane);
	const int t0 = r.first / KV_TILE + split * chunk;
	const int t1 = min(t0 + chunk, (max(r.last, 0) + KV_TILE - 1) / KV_TILE);
	if (split > 0 && t0 >= t1)
		return;

	/* the query row: its parts, and the sums that start the accumulators */
	half8_t qf[QP][L::G];
	float qsum[L::G], rs;
	{
		float v[L::G][8], top = 0.0f;
		const typename T::t *x = q + r.at * q_stride + (size_t)r.head * D;
#pragma unroll
		for (int g = 0; g < L::G; g++) {
			const kv_vec<TY, 8> w = *(const kv_vec<TY, 8> *)(x + 32 * g + 8 * part);
#pragma unroll
			for (int j = 0; j < 8; j++) {
				v[g][j] = T::get(w.v[j]);
				top = fmaxf(top, fabsf(v[g][j]));
			}
		}
		top = row_max(top);
		int e = 14 - exponent(top);
		e = top > 0.0f && top < __builtin_inff() ? min(max(e, -126), 126) : 0;
		const float sc = pow2(e);
		rs = scale * (1.44269504088896341f / KV_CODE_STEP) * pow2(-e);
#pragma unroll
		for (int g = 0; g < L::G; g++) {
			float sum = 0.0f;
#pragma unroll
			for (int j = 0; j < 8; j++) {
				const float y = v[g][j] * sc;
				const _Float16 hi = (_Float16)y;
				qf[0][g][j] = hi;
				sum += (float)hi;
				if (QP > 1) {
					const _Float16 lo = (_Float16)(y - (float)hi);
					qf[QP - 1][g][j] = lo;
					sum += (float)lo;
				}
			}
			qsum[g] = -8.0f * KV_CODE_STEP * row_sum(sum);
		}
	}

	floatx4 o[CT];
#pragma unroll
	for (int c = 0; c < CT; c++)
		o[c] = (floatx4)0.0f;
	float m = -__builtin_inff(), l = 0.0f;
	int pe = -1000; /* probabilities are multiplied by 2^pe; unset */

	for (int t = t0 + wave; t < t1; t += KV_WAVES) {
		const uint8_t *tile = kv_tile_at<D>(a, s, kv_head, t);
		if (!tile) {
			if (lane == 0)
				kv_error(a, HIP_KV_ERR_PAGE);
			continue;
		}
		float x[8], dv[8];
#pragma unroll
		for (int h = 0; h < 2; h++) {
			u32 kw[L::G];
			_Float16 kd[4][L::G];
#pragma unroll
			for (int g = 0; g < L::G; g++)
				kw[g] = ((const u32 *)tile)[((h * (L::G / L::P) + g / L::P) * 64 + lane) * L::P +
							     g % L::P];
#pragma unroll
			for (int j = 0; j < 4; j++) {
				const int row = 16 * h + 4 * part + j;
				dv[4 * h + j] = (float)((const _Float16 *)(tile + L::V_SCALES))[row];
#pragma unroll
				for (int g = 0; g < L::G; g++)
					kd[j][g] = ((const _Float16 *)(tile + L::K_SCALES))[row * L::G + g];
				x[4 * h + j] = 0.0f;
			}
#pragma unroll
			for (int g = 0; g < L::G; g++) {
				floatx4 acc = (floatx4)qsum[g];
				const half8_t kf = kv_word(kw[g], 0);
#pragma unroll
				for (int p = 0; p < QP; p++)
					acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[p][g], acc, 0, 0, 0);
#pragma unroll
				for (int j = 0; j < 4; j++)
					x[4 * h + j] = fmaf((float)kd[j][g], acc[j], x[4 * h + j]);
			}
		}
		const bool edge = t * KV_TILE < r.inner0 || (t + 1) * KV_TILE > r.inner1;
		float top = -__builtin_inff(), big = 0.0f;
#pragma unroll
		for (int j = 0; j < 8; j++) {
			x[j] *= rs;
			if (edge) {
				const int at = t * KV_TILE + 16 * (j / 4) + 4 * part + j % 4;
				if (at < r.lo || at >= r.hi)
					x[j] = -__builtin_inff();
				if (at < r.first || at >= r.last)
					dv[j] = 0.0f;
			}
			top = fmaxf(top, x[j]);
			big = fmaxf(big, fabsf(dv[j]));
		}
		top = fmaxf(m, row_max(top));
		const float base = top == -__builtin_inff() ? 0.0f : top;
		const float alpha = __builtin_amdgcn_exp2f(m - base);
		float back = alpha;
		m = top;
		/* the probabilities' scale: the same in all lanes, since the value
		 * scales are; lowered when a larger one comes */
		big = row_max(big);
		const int e = big > 0.0f ? 15 - exponent(big) : 100;
		if (pe == -1000) {
			pe = min(e, 100) - 1;
		} else if (e < pe) {
			back *= pow2(max(e - 1 - pe, -126));
			pe = e - 1;
		}
		const float ps = pow2(pe);
		float sum = 0.0f, w[8];
#pragma unroll
		for (int j = 0; j < 8; j++) {
			const float p = __builtin_amdgcn_exp2f(x[j] - base);
			sum += p;
			w[j] = edge && p == 0.0f ? 0.0f : p * (dv[j] * ps);
		}
		l = l * alpha + sum;
		half8_t pf[PP];
#pragma unroll
		for (int j = 0; j < 8; j++) {
			const _Float16 hi = (_Float16)w[j];
			pf[0][j] = hi;
			if (PP > 1)
				pf[PP - 1][j] = (_Float16)(w[j] - (float)hi);
		}
		if (__ballot(back != 1.0f)) {
#pragma unroll
			for (int c = 0; c < CT; c++)
				o[c] *= back;
		}
#pragma unroll
		for (int c = 0; c < CT; c++) {
			const u32 vw = ((const u32 *)(tile + L::V_CODES))[(c / 4 * 64 + lane) * 4 + c % 4];
			const half8_t vf = kv_word(vw, 0x4c004c00u) - (half8_t)(_Float16)24.0f;
#pragma unroll
			for (int p = 0; p < PP; p++)
				o[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[p], o[c], 0, 0, 0);
		}
	}

	/* the waves' results: to one maximum, then added in wave order */
	l = row_sum(l);
	if (part == 0) {
		s_m[wave][lane] = m;
		s_l[wave][lane] = l;
	}
	__syncthreads();
	float top = s_m[0][lane % 16];
#pragma unroll
	for (int w = 1; w < KV_WAVES; w++)
		top = fmaxf(top, s_m[w][lane % 16]);
	const float back = top == -__builtin_inff() ? 0.0f : top;
	float factor = pe == -1000 ? 0.0f : __builtin_amdgcn_exp2f(m - back) * pow2(-pe);
#pragma unroll
	for (int c = 0; c < CT; c++)
#pragma unroll
		for (int j = 0; j < 4; j++)
			s_o[wave][lane % 16][16 * c + 4 * part + j] = pe == -1000 ? 0.0f : o[c][j] * factor;
	__syncthreads();
	const size_t slot = ((size_t)(s * row_tiles + rt) * a.kv_heads + kv_head) * splits + split;
	for (int at = threadIdx.x; at < KV_ROWS * D / 4; at += KV_NT) {
		const int row = at / (D / 4), c = at % (D / 4) * 4;
		const kv_span z = kv_rows_of(sq, rt, G, kv_head, window, row);
		if (!z.valid)
			continue;
		float high = s_m[0][row], den = 0.0f, y[4] = {};
#pragma unroll
		for (int w = 1; w < KV_WAVES; w++)
			high = fmaxf(high, s_m[w][row]);
		const float zero = high == -__builtin_inff() ? 0.0f : high;
#pragma unroll
		for (int w = 0; w < KV_WAVES; w++) {
			den += s_l[w][row] * __builtin_amdgcn_exp2f(s_m[w][row] - zero);
#pragma unroll
			for (int u = 0; u < 4; u++)
				y[u] += s_o[w][row][c + u];
		}
		if (splits == 1) {
			kv_vec<TY, 4> v;
#pragma unroll
			for (int u = 0; u < 4; u++)
				v.v[u] = T::put(z.hi > z.lo ? y[u] / den : 0.0f);
			*(kv_vec<TY, 4> *)(out + z.at * out_stride + (size_t)z.head * D + c) = v;
			continue;
		}
		float *to = ws + slot * KV_ROWS * (D + 2);
		*(floatx4 *)(to + row * D + c) = floatx4{y[0], y[1], y[2], y[3]};
		if (c == 0) {
			to[KV_ROWS * D + 2 * row] = high;
			to[KV_ROWS * D + 2 * row + 1] = den;
		}
	}
}

/* the workgroups' results of one tile of query rows, added in their order */
template <int D, int TY>
__global__ __launch_bounds__(KV_NT) void k_kv_merge(kv_args a, int G, typename kv_type<TY>::t *out,
						     size_t out_stride, int window, const float *ws,
						     int row_tiles, int chunk, int splits)
{
	typedef kv_type<TY> T;
	int b = blockIdx.x;
	const int kv_head = b % a.kv_heads;
	b /= a.kv_heads;
	const int rt = b % row_tiles, s = b / row_tiles;
	const kv_seq sq = kv_sequence(a, s);
	if (rt * KV_ROWS >= sq.n * G)
		return;
	const float *part = ws + ((size_t)(s * row_tiles + rt) * a.kv_heads + kv_head) * splits *
					 KV_ROWS * (D + 2);
	for (int at = threadIdx.x; at < KV_ROWS * D / 4; at += KV_NT) {
		const int row = at / (D / 4), c = at % (D / 4) * 4;
		const kv_span z = kv_rows_of(sq, rt, G, kv_head, window, row);
		if (!z.valid)
			continue;
		const int tiles = (max(z.last, 0) + KV_TILE - 1) / KV_TILE - z.first / KV_TILE;
		const int n = min(splits, max(1, (tiles + chunk - 1) / chunk));
		float m = -__builtin_inff(), l = 0.0f;
		floatx4 y = (floatx4)0.0f;
		for (int i = 0; i < n; i++) {
			const float *p = part + (size_t)i * KV_ROWS * (D + 2);
			m = fmaxf(m, p[KV_ROWS * D + 2 * row]);
		}
		const float base = m == -__builtin_inff() ? 0.0f : m;
		for (int i = 0; i < n; i++) {
			const float *p = part + (size_t)i * KV_ROWS * (D + 2);
			const float f = __builtin_amdgcn_exp2f(p[KV_ROWS * D + 2 * row] - base);
			l += p[KV_ROWS * D + 2 * row + 1] * f;
			y += *(const floatx4 *)(p + row * D + c) * f;
		}
		kv_vec<TY, 4> v;
#pragma unroll
		for (int u = 0; u < 4; u++)
			v.v[u] = T::put(z.hi > z.lo ? y[u] / l : 0.0f);
		*(kv_vec<TY, 4> *)(out + z.at * out_stride + (size_t)z.head * D + c) = v;
	}
}

extern "C" void kv_attn_plan(const kv_args *a, int head_len, int heads, int window, kv_plan *p)
{
	const int G = heads / a->kv_heads;
	const long all = ((long)a->max_len + KV_TILE - 1) / KV_TILE;
	long tiles = all; /* of the cache that one tile of query rows sees, at most */
	if (window && (long)window + KV_ROWS < a->max_len)
		tiles = ((long)window + KV_ROWS + KV_TILE - 2) / KV_TILE + 1;
	tiles = tiles < all ? tiles : all;
	p->row_tiles = (int)(((long)a->max_rows * G + KV_ROWS - 1) / KV_ROWS);
	const size_t wgs = (size_t)a->nseq * a->kv_heads * p->row_tiles;
	/* along the cache: enough workgroups to fill the chip, each with a tile
	 * for every wave at least */
	const long want = wgs ? (long)((1024 + wgs - 1) / wgs) : 1;
	const long most = (all + KV_WAVES - 1) / KV_WAVES;
	const long splits = want < most ? want : most > 1 ? most : 1;
	long chunk = (tiles + splits - 1) / splits;
	chunk = (chunk + KV_WAVES - 1) / KV_WAVES * KV_WAVES;
	p->chunk = (int)(chunk < KV_WAVES ? KV_WAVES : chunk);
	p->splits = (int)((tiles + p->chunk - 1) / p->chunk);
	p->splits = p->splits < 1 ? 1 : p->splits;
	/* without regard to the window, so that one workspace serves any */
	p->ws = splits > 1 ? wgs * splits * KV_ROWS * (head_len + 2) * sizeof(float) : 0;
}

extern "C" int kv_launch_attn(const kv_args *a, int head_len, int type, const void *q,
			      size_t q_stride, int heads, void *out, size_t out_stride, float scale,
			      int window, void *ws, const kv_plan *p, void *stream)
{
	const int G = heads / a->kv_heads;
	const size_t wgs = (size_t)a->nseq * a->kv_heads * p->row_tiles;
	KV_DISPATCH_HEAD(head_len, D, KV_DISPATCH_TYPE(type, TY, {
		typedef kv_type<TY>::t t;
		k_kv_attn<D, TY><<<dim3((unsigned)(wgs * p->splits)), KV_NT, 0, (hipStream_t)stream>>>(
			*a, (const t *)q, q_stride, G, (t *)out, out_stride, scale, window, (float *)ws,
			p->row_tiles, p->chunk, p->splits);
		if (p->splits > 1)
			k_kv_merge<D, TY><<<dim3((unsigned)wgs), KV_NT, 0, (hipStream_t)stream>>>(
				*a, G, (t *)out, out_stride, window, (const float *)ws, p->row_tiles,
				p->chunk, p->splits);
	}))
	return (int)hipGetLastError();
}
