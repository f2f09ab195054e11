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
 * row's scale its probability.  How a code becomes f16 is at kv_word below.  The keys'
 * surplus of 8 a channel leaves through the accumulator's start (-8 sum of the query's
 * channels) or through a product of its own, the values' by a subtraction, exact as
 * well, since over many cached rows a surplus would outweigh the sum.  A query row is
 * scaled by a power of two and, from fp32, split into two f16 parts of together 22
 * bits; f16 and bf16 queries are exact in one.  The probability times the value scale
 * is scaled by a power of two that keeps it within f16, and split in two as well.  For
 * bf16 outputs one part is enough: it is rounded by 2^-11 at most, with no bias (the
 * denominator sums what was not rounded), where the output is rounded by up to 2^-8.
 * Sums, maxima and exponents are fp32.
 *
 * Three forms, chosen by kv_attn_plan: few rows in slots of columns and up to 16 rows
 * (k_kv_attn; HBM bounds long caches, latency short ones), and tiles of 32 rows for
 * prompts (k_kv_attn_wide; VALU: making f16 of codes, scales and exponentials take
 * three times the matrix instructions' cycles).
 */
#include "kv_device.h"

#include <type_traits>

#define KV_NT 256
#define KV_WAVES (KV_NT / WAVE)
#define KV_ROWS 16 /* query rows of a tile */
#define KV_SPLITS 1024 /* pieces of a cache, at most */

__device__ static inline half8_t as_half8(u32 a, u32 b, u32 c, u32 d)
{
	const u32x4 v = {a, b, c, d};
	return __builtin_bit_cast(half8_t, v);
}

/*
 * A word's codes as f16, in their order: a turn and four masks for eight.
 *
 * 16-bit types (kv_word): the bits where they lie and nothing around them,
 * subnormals: code * 2^-22 for codes 0, 1, 4 and 5, code * 2^-18 for the others; the
 * other operand has 16 times the value where the code has the smaller step.  The
 * matrix cores align products by the exponent that an operand has, not by its
 * leading bit, so that the smaller ones lose four bits of the sum's 24, more than
 * enough for outputs of 8 or 11 bits (3e-6 of the output's norm).
 *
 * fp32: all with the larger step (kv_word_even), for keys whose surplus of 8 is in the
 * accumulators' start; or with exponents that make both steps 1/16, 16 + code / 16
 * and 1 + code / 16, of which 16.5 and 1.5 leave (code - 8) / 16, normal and exact
 * (kv_word8): 4e-7.
 */
__device__ static inline half8_t kv_word(u32 w)
{
	const u32 r = kv_rotr(w, 8);
	return as_half8(w & 0x003c003cu, w & 0x03c003c0u, r & 0x003c003cu, r & 0x03c003c0u);
}

/* whether code j has the smaller step */
__device__ static constexpr bool kv_small(int j)
{
	return j % 4 < 2;
}

/* how a type's operands are made: the codes' step, the exponents of a query row's
 * largest value and of its largest probability times value scale (kv_soft below) */
template <int TY> struct kv_form {
	static constexpr bool EVEN = TY == HIP_KV_F32;
	static constexpr float KEY_STEP = 1.0f / (1 << 18); /* kv_word, kv_word_even */
	static constexpr float STEP = EVEN ? 1.0f / 16.0f : KEY_STEP; /* kv_word8 */
	static constexpr float MORE = EVEN ? 1.0f : 16.0f; /* where the codes have the smaller step */
	static constexpr int QUERY = EVEN ? 14 : 10;
	static constexpr float LOG_MORE = EVEN ? 0.0f : 4.0f;
	static constexpr float REF = EVEN ? 9.0f : 5.0f, TOP = EVEN ? 15.0f : 11.0f;
};

/* all codes with the larger step */
__device__ static inline half8_t kv_word_even(u32 w)
{
	const u32 m = 0x03c003c0u;
	return as_half8(w << 4 & m, w & m, w >> 4 & m, kv_rotr(w, 8) & m);
}

/* 8 in the steps of kv_word's codes */
__device__ static inline half8_t kv_surplus8()
{
	const _Float16 a = (_Float16)(8.0f / (1 << 22)), b = (_Float16)(8.0f / (1 << 18));
	return half8_t{a, a, b, b, a, a, b, b};
}

/* (the compiler takes two instructions for want of a second scalar operand) */
__device__ static inline u32 and_or(u32 x, u32 mask, u32 bits)
{
	u32 y;
	asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(y) : "v"(x), "s"(mask), "v"(bits));
	return y;
}

/* the codes less 8 */
template <int TY> __device__ static inline half8_t kv_word8(u32 w)
{
	if constexpr (!kv_form<TY>::EVEN)
		return kv_word(w) - kv_surplus8();
	const u32 r = kv_rotr(w, 8), m = 0x003c003cu, n = 0x03c003c0u, sixteen = 0x4c004c00u, one = 0x3c003c00u;
	const _Float16 a = (_Float16)16.5f, b = (_Float16)1.5f;
	return as_half8(and_or(w, m, sixteen), and_or(w, n, one), and_or(r, m, sixteen), and_or(r, n, one)) -
	       half8_t{a, a, b, b, a, a, b, b};
}

/* x = hi + lo in f16; the products with the hidden -1 stay fused with the
 * conversions */
__device__ static inline _Float16 rest(float x, _Float16 hi)
{
	float minus = -1.0f;
	asm("" : "+s"(minus));
	return (_Float16)fmaf((float)hi, minus, x);
}

/* v and its copy after an exchange of the odd rows of 16 lanes (SPAN 16; the
 * upper 32 lanes, SPAN 32) of the one with the even rows (the lower) of the other:
 * both lanes of a pair that far apart then hold both of their values */
template <int SPAN> __device__ static inline float2 swapped(float v)
{
	const u32 u = __builtin_bit_cast(u32, v);
	const auto t = SPAN == 16 ? __builtin_amdgcn_permlane16_swap(u, u, false, false)
				  : __builtin_amdgcn_permlane32_swap(u, u, false, false);
	const u32 x = t[0], y = t[1];
	return make_float2(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y));
}

/* the largest (the sum) over the four lanes l % 16 that share a query row */
__device__ static inline float row_max(float v)
{
	float2 t = swapped<16>(v);
	t = swapped<32>(fmaxf(t.x, t.y));
	return fmaxf(t.x, t.y);
}

__device__ static inline float row_sum(float v)
{
	float2 t = swapped<16>(v);
	t = swapped<32>(t.x + t.y);
	return t.x + t.y;
}

/* the same of the two lanes l % 32 */
__device__ static inline float half_max(float v)
{
	const float2 t = swapped<32>(v);
	return fmaxf(t.x, t.y);
}

__device__ static inline float half_sum(float v)
{
	const float2 t = swapped<32>(v);
	return t.x + t.y;
}

/* 2^n, n within -126 .. 127 */
__device__ static inline float pow2(int n)
{
	return __builtin_bit_cast(float, (u32)(n + 127) << 23);
}

/* 2^(x - ref), 0 for a maximum (x or ref) that nothing was seen for */
__device__ static inline float weight(float x, float ref)
{
	return __builtin_amdgcn_exp2f(x - (ref == -__builtin_inff() ? 0.0f : ref));
}

/* the cached rows that the lane's query row sees, and the tile's rows */
struct kv_span {
	int lo, hi;         /* of the lane's query row */
	int first, last;    /* of some row of the tile */
	int inner0, inner1; /* of every row of the tile */
	int row, head;      /* the row among the batch's rows, and its head */
	bool valid;
};

template <int ROWS, int SLOTS = 1>
__device__ static inline kv_span kv_rows_of(const kv_seq &sq, int tile, int G, int kv_head, int window,
					    int lane)
{
	kv_span r;
	const int base = sq.len - sq.n, all = sq.n * G;
	const int mine = tile * ROWS + lane % (ROWS * SLOTS) / SLOTS, kept = min(mine, all - 1), i = kept / G;
	const int i0 = __builtin_amdgcn_readlane(i, 0), i1 = __builtin_amdgcn_readlane(i, ROWS * SLOTS - 1);
	r.valid = mine < all;
	r.hi = base + i + 1;
	r.lo = window ? max(0, r.hi - window) : 0;
	r.row = sq.row + i;
	r.head = kv_head * G + kept - i * G;
	r.last = base + i1 + 1;
	r.first = window ? max(0, base + i0 + 1 - window) : 0;
	r.inner0 = window ? max(0, r.last - window) : 0;
	r.inner1 = base + i0 + 1;
	return r;
}

/* a tile of the cache in registers: the lane's share, as the layout has it */
template <int D> struct kv_keys {
	typedef kv_tile<D> L;
	u32 w[2][L::G];        /* rows lane % 16 of each half */
	u32x4 d[2][L::G / 2];  /* scales of rows 4 (lane / 16) + j of each half */
	__device__ inline float scale(int h, int j, int g) const
	{
		return (float)__builtin_bit_cast(half8_t, d[h][(j * L::G + g) / 8])[(j * L::G + g) % 8];
	}
	/* the one of two or four from word u on whose bytes pick names */
	__device__ inline float scale_of(int h, int u, int n, u32 pick) const
	{
		const u32 lo = d[h][u / 4][u % 4], hi = n > 2 ? d[h][u / 4][u % 4 + 1] : lo;
		return (float)__builtin_bit_cast(half2_t, __builtin_amdgcn_perm(hi, lo, pick))[0];
	}
	__device__ inline void load(const uint8_t *tile, int lane)
	{
#pragma unroll
		for (int h = 0; h < 2; h++) {
			typedef uint32_t words __attribute__((ext_vector_type(L::P)));
#pragma unroll
			for (int g = 0; g < L::G; g += L::P) {
				const words x = ((const words *)tile)[(h * (L::G / L::P) + g / L::P) * 64 + lane];
#pragma unroll
				for (int u = 0; u < L::P; u++)
					w[h][g + u] = x[u];
			}
			const u32x4 *s = (const u32x4 *)(tile + L::K_SCALES) + (16 * h + 4 * (lane / 16)) * L::G / 8;
#pragma unroll
			for (int u = 0; u < L::G / 2; u++)
				d[h][u] = s[u];
		}
	}
};

template <int D> struct kv_values {
	typedef kv_tile<D> L;
	u32 w[D / 16]; /* channels 16 c + lane % 16 */
	__device__ inline void load(const uint8_t *tile, int lane)
	{
		const u32x4 *p = (const u32x4 *)(tile + L::V_CODES) + lane;
#pragma unroll
		for (int c = 0; c < D / 64; c++) {
			const u32x4 x = p[64 * c];
#pragma unroll
			for (int u = 0; u < 4; u++)
				w[4 * c + u] = x[u];
		}
	}
};

/* value scales of the lane's rows: two or four of its eight with slots */
template <int SLOTS> struct kv_dv {
	u32 w[4 / SLOTS];
	__device__ inline void load(const uint8_t *scales, int lane)
	{
		const int c = lane % SLOTS, part = lane / 16;
		if constexpr (SLOTS == 4) {
			w[0] = ((const u32 *)scales)[8 * (c / 2) + 2 * part + c % 2];
		} else {
#pragma unroll
			for (int h = 0; h < 2 / SLOTS; h++) {
				const u32x2 a = ((const u32x2 *)scales)[4 * (SLOTS == 2 ? c : h) + part];
				w[2 * h] = a.x;
				w[2 * h + 1] = a.y;
			}
		}
	}
};

/*
 * A tile of query rows as the products take it, in LDS for all waves: part p of
 * group g of the lane's row at f[p][g][lane], and what the accumulators start
 * with, -8 steps times the groups' sum.
 */
template <int D, int QP, int SLOTS> struct kv_query {
	half8_t f[QP][D / 32][WAVE];
	floatx4 start[D / 32 / SLOTS][16];
};

/* what a query row whose largest value is top is multiplied by, and its scores
 * then, to be logits in powers of two (the latter a normal number whatever the scale:
 * a score of 0 or minus infinity stays what it is) */
struct kv_factor {
	float query, score;
};

template <int TY> __device__ static inline kv_factor kv_query_factor(float top, float scale, float key_step)
{
	int e = kv_form<TY>::QUERY - __builtin_amdgcn_frexp_expf(top);
	e = top > 0.0f && top < __builtin_inff() ? min(max(e, -126), 122) : 0;
	/* a negative scale turns the query around, 0 makes it 0 */
	const float score = (scale == 0.0f ? 1.0f : fabsf(scale)) * (1.44269504088896341f / key_step) * pow2(-e);
	return {scale > 0.0f ? pow2(e) : scale < 0.0f ? -pow2(e) : 0.0f, fminf(fmaxf(score, 0x1p-126f), 0x1.fffffep127f)};
}

/* eight channels of a query row in f16 parts, and their sum */
template <int QP, int TY>
__device__ static inline float kv_split8(const kv_vec<TY, 8> &w, float factor, half8_t (&f)[QP])
{
	float sum = 0.0f;
#pragma unroll
	for (int j = 0; j < 8; j++) {
		const float y = kv_type<TY>::get(w.v[j]) * (kv_small(j) ? kv_form<TY>::MORE * factor : factor);
		float z = (float)(f[0][j] = (_Float16)y);
		if (QP > 1)
			z += (float)(f[QP - 1][j] = rest(y, f[0][j]));
		sum += kv_small(j) ? z * (1.0f / kv_form<TY>::MORE) : z;
	}
	return sum;
}

/* The groups g % waves == wave of a tile of query rows into LDS, from w, the lane's
 * quarter of each group of its row; returns the scores' factor.  The caller
 * synchronises. */
template <int D, int QP, int SLOTS, int TY>
__device__ static inline float kv_put_query(kv_query<D, QP, SLOTS> &q, const kv_vec<TY, 8> (&w)[D / 32],
					    float scale, int lane, int wave, int waves)
{
	float top = 0.0f;
#pragma unroll
	for (int g = 0; g < D / 32; g++)
#pragma unroll
		for (int j = 0; j < 8; j++)
			top = fmaxf(top, fabsf(kv_type<TY>::get(w[g].v[j])));
	const kv_factor f = kv_query_factor<TY>(row_max(top), scale, kv_form<TY>::KEY_STEP);
#pragma unroll
	for (int g = 0; g < D / 32; g++) {
		if (g % waves != wave)
			continue;
		const bool own = lane % SLOTS == g % SLOTS;
		half8_t z[QP];
		const float start = -8.0f * kv_form<TY>::KEY_STEP * row_sum(kv_split8<QP, TY>(w[g], f.query, z));
#pragma unroll
		for (int p = 0; p < QP; p++)
			q.f[p][g][lane] = own ? z[p] : (half8_t)(_Float16)0.0f;
		if (own && lane < 16)
			q.start[g / SLOTS][lane] = (floatx4)start;
	}
	return f.score;
}

/* v of the lane whose number differs in the bit BY, 1 or 2 */
template <int BY> __device__ static inline float other(float v)
{
	/* quad_perm 1 0 3 2, 2 3 0 1 */
	return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), BY == 1 ? 0xb1 : 0x4e,
								  0xf, 0xf, true));
}

/* the sums of v[N] over the lane and the one beside it: the lower lane's are the
 * first half, the upper's the second */
template <int BY, int N> __device__ static inline void halved(const float (&v)[N], bool upper, float *out)
{
#pragma unroll
	for (int i = 0; i < N / 2; i++) {
		const float mine = upper ? v[N / 2 + i] : v[i], theirs = upper ? v[i] : v[N / 2 + i];
		out[i] = mine + other<BY>(theirs);
	}
}

/* Scores of the lane's 8 / SLOTS cached rows: of 4 part + j of each half, j < 4, the
 * share of the lane's slot. */
template <int D, int QP, int SLOTS, int TY>
__device__ static inline auto kv_scores(const kv_keys<D> &k, const kv_query<D, QP, SLOTS> &q, int lane)
{
	typedef float floats __attribute__((ext_vector_type(8 / SLOTS)));
	constexpr int G = D / 32, NA = G / SLOTS; /* groups, and of a slot */
	const u32 b = 2 * (lane % SLOTS), pick = b | (b + 1) << 8 | 0x0c0c0000u;
	floats x;
	float y[8];
#pragma unroll
	for (int a = 0; a < NA; a++) {
		const floatx4 start = q.start[a][lane % 16];
		floatx4 acc[2] = {start, start};
#pragma unroll
		for (int g = a * SLOTS; g < (a + 1) * SLOTS; g++) {
			half8_t f[QP];
#pragma unroll
			for (int p = 0; p < QP; p++)
				f[p] = q.f[p][g][lane];
#pragma unroll
			for (int h = 0; h < 2; h++) {
				const half8_t kf = kv_form<TY>::EVEN ? kv_word_even(k.w[h][g]) : kv_word(k.w[h][g]);
#pragma unroll
				for (int p = 0; p < QP; p++)
					acc[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, f[p], acc[h], 0, 0, 0);
			}
		}
#pragma unroll
		for (int h = 0; h < 2; h++)
#pragma unroll
			for (int j = 0; j < 4; j++) {
				const int at = 4 * h + j;
				const float d = SLOTS == 1 ? k.scale(h, j, a) : k.scale_of(h, (j * G + a * SLOTS) / 2, SLOTS, pick);
				y[at] = fmaf(d, acc[h][j], a ? y[at] : 0.0f);
			}
	}
	if constexpr (SLOTS == 4) {
		float t[4];
		halved<2>(y, lane & 2, t);
		halved<1>(t, lane & 1, y);
	} else if constexpr (SLOTS == 2) {
		float t[4];
		halved<1>(y, lane & 1, t);
#pragma unroll
		for (int j = 0; j < 4; j++)
			y[j] = t[j];
	}
#pragma unroll
	for (int j = 0; j < 8 / SLOTS; j++)
		x[j] = y[j];
	return x;
}

/*
 * The running softmax of a query row.  ref is its reference in powers of two: a
 * probability is 2^(logit - ref), and ref the largest sum of a logit and its value
 * scale's exponent, less REF, so that probability times value scale stays below
 * 2^REF and the largest is at least 2^(REF - 1 - SPREAD): the f16 parts hold the others
 * relative to it.  ref stays as it is until a product would reach 2^TOP (2^15 with
 * kv_word's factor, below f16's largest): most tiles then leave the output alone.
 * Sums and outputs carry the same factor, which the division at the end takes out.
 *
 * That sum's bound is the lane's largest logit plus its largest exponent.  They may be
 * different rows': where the bound would move ref and the lane's scales are 2^SPREAD
 * apart, subnormal or 0, it is taken row by row.  (Row by row always: 900 -> 950 us for the prompt
 * at k_kv_attn_wide.)  A row without a value (scale 0) then counts with the exponent
 * NO_VALUE: it moves ref only where its logit is far above all that has a value, and
 * its probability stays below 2^(TOP - NO_VALUE), of which fp32 holds the sum of 2^31.
 */
struct kv_soft {
	float ref, sum;
	static constexpr int SPREAD = 8;
	static constexpr float NO_VALUE = -80.0f;
};

template <int N> using kv_halves = _Float16 __attribute__((ext_vector_type(N)));

/*
 * Probabilities times value scales of the lane's N cached rows, in f16 parts;
 * 16 times that where the codes have the smaller step: two of four rows, or (N = 2)
 * both of a lane with more = 4.  SPAN lanes 16 apart, or two 32 apart, hold the query
 * row's others.  rescale(f) multiplies the output so far, where the reference moves.
 */
template <int N, int SPAN, int PP, int TY, class Fn>
__device__ static inline void kv_softmax(kv_soft &s, const float *x, const half2_t *dv, float rs, float more,
					 kv_halves<N> (&pf)[PP], Fn rescale)
{
	constexpr float LOG_MORE = kv_form<TY>::LOG_MORE, MORE = kv_form<TY>::MORE;
	float top = x[0];
#pragma unroll
	for (int j = 1; j < N; j++)
		top = fmaxf(top, x[j]);
	/* f16 without their sign order as whole numbers do */
	ushort2_t most2 = {0, 0};
#pragma unroll
	for (int i = 0; i < N / 2; i++) {
		const u32 a = __builtin_bit_cast(u32, dv[i]) & 0x7fff7fffu;
		most2 = __builtin_elementwise_max(most2, __builtin_bit_cast(ushort2_t, a));
	}
	const unsigned short most1 = most2.x > most2.y ? most2.x : most2.y;
	const float big = (float)__builtin_bit_cast(_Float16, most1);
	/* (scales of nothing but zeros: exponent 0, and row by row below) */
	const float most = fmaf(top, rs, (float)__builtin_amdgcn_frexp_expf(big));
	float high = SPAN == 4 ? row_max(most) : half_max(most);
	float next = high - s.ref > kv_form<TY>::TOP ? high - kv_form<TY>::REF : s.ref;
	float back = weight(s.ref, next);
	if (__ballot(back != 1.0f)) {
		ushort2_t least2 = {0xffff, 0xffff};
#pragma unroll
		for (int i = 0; i < N / 2; i++) {
			const u32 a = __builtin_bit_cast(u32, dv[i]) & 0x7fff7fffu;
			least2 = __builtin_elementwise_min(least2, __builtin_bit_cast(ushort2_t, a));
		}
		const unsigned short least1 = least2.x < least2.y ? least2.x : least2.y;
		if (__ballot(least1 < 1 << 10 || most1 - least1 > kv_soft::SPREAD << 10)) {
			float own = -__builtin_inff();
#pragma unroll
			for (int j = 0; j < N; j++) {
				const float d = (float)dv[j / 2][j % 2];
				own = fmaxf(own, fmaf(x[j], rs, d == 0.0f ? kv_soft::NO_VALUE
									  : (float)__builtin_amdgcn_frexp_expf(d)));
				asm("" : "+v"(own)); /* (few registers) */
			}
			high = SPAN == 4 ? row_max(own) : half_max(own);
			next = high - s.ref > kv_form<TY>::TOP ? high - kv_form<TY>::REF : s.ref;
			back = weight(s.ref, next);
		}
		rescale(back);
	}
	s.ref = next;
	const float ref = next == -__builtin_inff() ? 0.0f : next;
	const float ref16 = N == 2 && LOG_MORE > 0.0f ? ref - more : ref - LOG_MORE;
	float sum = 0.0f, sum16 = 0.0f;
#pragma unroll
	for (int j = 0; j < N; j++) {
		const float p = __builtin_amdgcn_exp2f(fmaf(x[j], rs, kv_small(j) ? -ref16 : -ref));
		(kv_small(j) ? sum16 : sum) += p;
		float w = fmaf((float)dv[j / 2][j % 2], p, 0.0f); /* fma: takes an f16 as it is */
		if (PP > 1)
			asm("" : "+v"(w)); /* once, not once for each part */
		pf[0][j] = (_Float16)w;
		if (PP > 1)
			pf[PP - 1][j] = rest(w, pf[0][j]);
	}
	const float less = N == 2 && more == 0.0f ? 1.0f : 1.0f / MORE;
	s.sum = s.sum * back + fmaf(sum16, less, sum);
}

/*
 * The caches of a call with one row tile a sequence as one line of tiles, sequence
 * after sequence, cut into equal shares: of this workgroup's sequences (a thread
 * each, KV_SEQS at most) where they start in it, and the whole line's length.  A
 * sequence with rows has a tile at least.
 */
#define KV_SEQS KV_NT

struct kv_line {
	int start, tiles; /* of sequence threadIdx.x */
	int all;
};

__device__ static inline kv_line kv_line_of(const kv_args &a, int window)
{
	__shared__ int s_wave[KV_WAVES];
	const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
	int tiles = 0;
	if ((int)threadIdx.x < a.nseq) {
		const kv_seq sq = kv_sequence(a, threadIdx.x, true);
		const int first = window ? max(0, sq.len - sq.n + 1 - window) : 0;
		tiles = sq.n ? max(1, (max(sq.len, 0) + KV_TILE - 1) / KV_TILE - first / KV_TILE) : 0;
	}
	int end = tiles;
	for (int o = 1; o < WAVE; o <<= 1) {
		const int before = __shfl_up(end, o, WAVE);
		end += lane >= o ? before : 0;
	}
	if (lane == WAVE - 1)
		s_wave[wave] = end;
	__syncthreads();
	kv_line r = {end - tiles, tiles, 0};
#pragma unroll
	for (int w = 0; w < KV_WAVES; w++) {
		r.start += w < wave ? s_wave[w] : 0;
		r.all += s_wave[w];
	}
	return r;
}

/* tiles of each of n shares */
__device__ static inline int kv_share(int all, int n)
{
	return max((all + n - 1) / n, KV_WAVES);
}

/*
 * Few query rows: one workgroup takes a tile of them over `chunk` tiles of the
 * cache, dealt to its waves one by one; the waves' results meet in LDS.
 * With more than one workgroup along the cache each leaves its reference, sum
 * and unnormalised output in ws for k_kv_merge.  A wave loads a tile's keys
 * while it still works on the values of the tile before, and the values while
 * it works on the keys.
 *
 * SLOTS columns of the products belong to one query row where there are few, four
 * for rows up to 4 (heads of 128 and 256), two for up to 8.  In the first product a
 * slot has its share of the channel groups and zeros for the others: the partial
 * scores of a row's groups come out in different lanes, which multiply them by their
 * own scales, add up and keep 8 / SLOTS of the cached rows each (scale products and
 * exponentials a row: 8 and 2 instead of 32 and 8 for four slots).  In the second
 * product a slot has its cached rows and zeros for the others; its statistics and
 * output are its own, like another wave's, until the end.
 *
 * SHARE: instead of a piece of one cache the workgroup has an equal share of all of
 * them, one after the other, and takes the sequences in it in turn.
 *
 * 131072 rows, 32 bf16 heads on 8 of 128 (145 MB): 31.8 us and the merge 4.2, 4.1 TB/s
 * in all; without slots 34.9.  64 sequences of 340 to 16384 rows in fp32 (341 MB):
 * 88 us with the merge, 3.9 TB/s; in pieces 97.5, without slots and at three waves a
 * SIMD 118.
 */
/* by the registers: four waves a SIMD with slots, which is two workgroups of KV_MANY a
 * CU (64 sequences x 2300 rows, 32 fp32 heads on 8: 37.9 us; with two registers too many
 * for that 41.9), three without, two for heads of 256.  Nothing is kept in accumulation
 * registers and moved. */
template <int D, int TY, int NW, int SLOTS, bool SHARE>
__global__ __launch_bounds__(NW * WAVE) __attribute__((amdgpu_waves_per_eu(D == 256 ? 2 : SLOTS > 1 ? 4 : 3)))
void k_kv_attn(
	kv_args a, const typename kv_type<TY>::t *q, size_t q_stride, int G,
	typename kv_type<TY>::t *out, size_t out_stride, float scale, int window, float *ws,
	int row_tiles, int chunk, int nrows)
{
	typedef kv_type<TY> T;
	typedef kv_tile<D> L;
	constexpr int QP = TY == HIP_KV_F32 ? 2 : 1, PP = TY == HIP_KV_BF16 ? 1 : 2;
	constexpr int CT = D / 16; /* channel tiles of O^T */
	constexpr int ROWS = KV_ROWS / SLOTS, N = 8 / SLOTS;
	/* the queries, then the waves' outputs */
	__shared__ union {
		kv_query<D, QP, SLOTS> q;
		float o[NW][ROWS][D + 4];
	} sh;
	__shared__ float s_ref[NW][KV_ROWS], s_sum[NW][ROWS], s_high[ROWS];
	__shared__ int s_row[ROWS], s_head[ROWS], s_seq[2];
	__shared__ int2 s_line[SHARE ? KV_SEQS : 1]; /* a sequence's start and tiles in the line */

	const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
	const int kv_head = blockIdx.x % a.kv_heads, rt = blockIdx.x / a.kv_heads;
	const int split = blockIdx.y, splits = gridDim.y, shift = a.page_shift - 5;
	int pos = 0, end = 1; /* of the workgroup's share of the line */
	if constexpr (SHARE) {
		const kv_line line = kv_line_of(a, window);
		s_line[threadIdx.x] = make_int2(line.start, line.tiles);
		const int share = kv_share(line.all, splits);
		pos = split * share;
		end = min(pos + share, line.all);
	}
	while (pos < end) {
		int lane = threadIdx.x % WAVE;
		if constexpr (SHARE) { /* nothing of the lane's is kept in registers from turn to turn */
			asm volatile("" : "+v"(lane));
			__builtin_assume(lane >= 0 && lane < WAVE);
		}
		const int part = lane / 16, slot = lane % SLOTS;
		int s = blockIdx.z, t0 = 0, t1 = 0, page = -1;
		if constexpr (SHARE) {
			const int2 line = s_line[threadIdx.x];
			if (line.x <= pos && pos < line.x + line.y) {
				s_seq[0] = threadIdx.x;
				s_seq[1] = line.x;
			}
			__syncthreads();
			s = __builtin_amdgcn_readfirstlane(s_seq[0]);
			t0 = pos - __builtin_amdgcn_readfirstlane(s_seq[1]);
		}
		/* the wave's tiles t0 + wave, + NW, ..; a lane holds the page of one of the
		 * next 64.  Without a window the first lot needs no length, only the table's
		 * bound, and is on its way before the length is known */
		const int32_t *table = a.table + s * a.table_stride;
		if (!window && !SHARE) {
			const int at = (split * chunk + wave + lane * NW) >> shift;
			page = at < a.table_stride ? table[at] : -1;
		}
		const kv_seq sq = kv_sequence(a, s);
		if (!SHARE && rt * ROWS >= sq.n * G)
			return;
		const kv_span r = kv_rows_of<ROWS, SLOTS>(sq, rt, G, kv_head, window, lane);
		t1 = (max(r.last, 0) + KV_TILE - 1) / KV_TILE;
		if constexpr (SHARE) {
			t0 += r.first / KV_TILE;
			const int take = max(1, min(end - pos, t1 - t0));
			t1 = min(t1, t0 + take);
			pos += take;
		} else {
			t0 = r.first / KV_TILE + split * chunk;
			t1 = min(t0 + chunk, t1);
			pos = end;
			if (split > 0 && t0 >= t1)
				return;
		}
		kv_vec<TY, 8> qv[L::G];
#pragma unroll
		for (int g = 0; g < L::G; g++)
			qv[g] = *(const kv_vec<TY, 8> *)(q + (size_t)r.row * q_stride + (size_t)r.head * D + 32 * g + 8 * part);

		/* (a page outside the pool: its first tile, with every row hidden) */
		const int n = a.pages ? (t1 - t0 - wave + NW - 1) / NW : 0;
		bool lost = false;
		const auto tile_of = [&](int i) -> const uint8_t * {
			const int t = t0 + wave + i * NW;
			if (i % WAVE == 0 && (i || window || SHARE)) {
				const int tl = t + lane * NW;
				page = tl < t1 ? table[tl >> shift] : -1;
			}
			const int id = __builtin_amdgcn_readlane(page, i % WAVE);
			lost = (u32)id >= (u32)a.pages;
			const size_t at = lost ? 0 : ((((size_t)id * a.kv_heads + kv_head) << shift) + (t & ((1 << shift) - 1)));
			return a.pool + at * L::BYTES;
		};
		kv_keys<D> k;
		kv_values<D> v;
		kv_dv<SLOTS> vd;
		if (n > 0) {
			const uint8_t *tile = tile_of(0);
			k.load(tile, lane);
			vd.load(tile + L::V_SCALES, lane);
			v.load(tile, lane);
		} else if (!a.pages && t1 > t0 && lane == 0) {
			kv_error(a, HIP_KV_ERR_PAGE);
		}
		const float rs = kv_put_query<D, QP, SLOTS, TY>(sh.q, qv, scale, lane, wave, NW);
		if (threadIdx.x < KV_ROWS && slot == 0) {
			s_row[threadIdx.x / SLOTS] = r.valid ? r.row : -1;
			s_head[threadIdx.x / SLOTS] = r.hi > r.lo ? r.head : ~r.head;
		}
		__syncthreads();

		floatx4 o[CT];
#pragma unroll
		for (int c = 0; c < CT; c++)
			o[c] = (floatx4)0.0f;
		kv_soft soft = {-__builtin_inff(), 0.0f};

		const auto step = [&](int i, auto more) {
			const int t = t0 + wave + i * NW;
			const bool hidden = lost;
			const uint8_t *next = NULL;
			if constexpr (more.value)
				next = tile_of(i + 1);
			half2_t dv[N / 2];
			kv_halves<N> pp[PP];
#pragma unroll
			for (int j = 0; j < N / 2; j++)
				dv[j] = __builtin_bit_cast(half2_t, vd.w[j]);
			typedef float floats __attribute__((ext_vector_type(N)));
			floats x = kv_scores<D, QP, SLOTS, TY>(k, sh.q, lane);
			/* the scales are used up before their registers are loaded again */
			asm volatile("" : "+v"(x) : : "memory");
			if constexpr (more.value)
				k.load(next, lane);
			if (hidden || t * KV_TILE < r.inner0 || (t + 1) * KV_TILE > r.inner1) {
				const int lo = hidden ? 0x7fffffff : r.lo;
#pragma unroll
				for (int j = 0; j < N; j++) {
					const int u = slot * N + j, at = t * KV_TILE + 16 * (u / 4) + 4 * part + u % 4;
					const bool hide = at < lo || at >= r.hi;
					x[j] = hide ? -__builtin_inff() : x[j];
					dv[j / 2][j % 2] = hide ? (_Float16)0.0f : dv[j / 2][j % 2];
				}
				if (hidden && lane == 0)
					kv_error(a, HIP_KV_ERR_PAGE);
			}
			kv_softmax<N, 4, PP, TY>(soft, (const float *)&x, dv, rs, slot % 2 ? 0.0f : 4.0f, pp, [&](float back) {
#pragma unroll
				for (int c = 0; c < CT; c++)
					o[c] *= back;
			});
			/* a slot's column has its rows alone */
			half8_t pf[PP];
#pragma unroll
			for (int p = 0; p < PP; p++) {
				if constexpr (SLOTS == 1) {
					pf[p] = pp[p];
				} else {
					typedef u32 words __attribute__((ext_vector_type(N / 2)));
					const words z = __builtin_bit_cast(words, pp[p]);
					u32 w[4];
#pragma unroll
					for (int u = 0; u < 4; u++)
						w[u] = u / (N / 2) == slot ? z[u % (N / 2)] : 0;
					pf[p] = as_half8(w[0], w[1], w[2], w[3]);
				}
			}
#pragma unroll
			for (int c = 0; c < CT; c++) {
				const half8_t vf = kv_word8<TY>(v.w[c]);
#pragma unroll
				for (int p = 0; p < PP; p++)
					o[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[p], o[c], 0, 0, 0);
			}
			if constexpr (more.value) {
				vd.load(next + L::V_SCALES, lane);
				v.load(next, lane);
			}
		};
		for (int i = 0; i < n - 1; i++)
			step(i, std::true_type());
		if (n > 0)
			step(n - 1, std::false_type());

		/* the waves' results: to one reference, then added in wave order */
		float sum = kv_form<TY>::STEP * row_sum(soft.sum); /* the outputs' own factor */
		if (part == 0)
			s_ref[wave][lane] = soft.ref;
		__syncthreads();
		float ref = -__builtin_inff(); /* of the row, whichever column */
#pragma unroll
		for (int w = 0; w < NW; w++)
#pragma unroll
			for (int c = 0; c < SLOTS; c++)
				ref = fmaxf(ref, s_ref[w][lane % 16 - slot + c]);
		const float factor = weight(soft.ref, ref);
		const int row = lane % 16 / SLOTS;
		sum *= factor;
		float y[4 * CT], z[2 * CT]; /* the row's slots added: each keeps its share of the channels */
#pragma unroll
		for (int u = 0; u < 4 * CT; u++)
			y[u] = o[u / 4][u % 4] * factor;
		if constexpr (SLOTS == 4) {
			sum += other<2>(sum);
			halved<2>(y, lane & 2, z);
#pragma unroll
			for (int u = 0; u < 2 * CT; u++)
				y[u] = z[u];
		}
		if constexpr (SLOTS > 1) {
			float w[8 * CT / SLOTS];
#pragma unroll
			for (int u = 0; u < 8 * CT / SLOTS; u++)
				w[u] = y[u];
			sum += other<1>(sum);
			halved<1>(w, lane & 1, y);
		}
		if (r.valid) {
#pragma unroll
			for (int u = 0; u < CT / SLOTS; u++)
				*(floatx4 *)&sh.o[wave][row][16 * (slot * (CT / SLOTS) + u) + 4 * part] =
					floatx4{y[4 * u], y[4 * u + 1], y[4 * u + 2], y[4 * u + 3]};
			if (part == 0 && slot == 0) {
				s_sum[wave][row] = sum;
				s_high[row] = ref; /* (every wave's the same) */
			}
		}
		__syncthreads();
		const size_t piece = SHARE ? (size_t)kv_head * (splits + a.nseq) + split + s
					   : ((size_t)(s * row_tiles + rt) * a.kv_heads + kv_head) * splits + split;
		float *to = ws + piece * nrows * (D + 4);
		for (int at = threadIdx.x; at < ROWS * D / 4; at += NW * WAVE) {
			const int i = at / (D / 4), c = at % (D / 4) * 4, row = s_row[i];
			if (row < 0)
				break; /* the rows behind are not there either */
			float den = s_sum[0][i];
			floatx4 y = *(const floatx4 *)&sh.o[0][i][c];
#pragma unroll
			for (int w = 1; w < NW; w++) {
				den += s_sum[w][i];
				y += *(const floatx4 *)&sh.o[w][i][c];
			}
			if (!SHARE && splits == 1) {
				kv_vec<TY, 4> z;
				const int head = s_head[i];
#pragma unroll
				for (int u = 0; u < 4; u++)
					z.v[u] = T::put(head >= 0 ? y[u] / den : 0.0f);
				*(kv_vec<TY, 4> *)(out + row * out_stride + (size_t)(head < 0 ? ~head : head) * D + c) = z;
				continue;
			}
			*(floatx4 *)(to + i * (D + 4) + c) = y;
			if (c == 0) {
				to[i * (D + 4) + D] = s_high[i];
				to[i * (D + 4) + D + 1] = den;
			}
		}
		if constexpr (SHARE)
			__syncthreads();
	}
}

/*
 * The pieces' results of one query row: first their weights, then D / 4 threads
 * take the row's channels, KV_NT / (D / 4) times over, each its share of the
 * pieces.  Two dependent reads: 4.2 us for 64 pieces of 32 rows.
 */
template <int D, int TY>
__global__ __launch_bounds__(KV_NT) void k_kv_merge(kv_args a, int G, typename kv_type<TY>::t *out,
						     size_t out_stride, int window, const float *ws,
						     int row_tiles, int chunk, int splits, int nrows, int shares)
{
	typedef kv_type<TY> T;
	constexpr int CH = D / 4, PARTS = KV_NT / CH;
	__shared__ floatx4 s_y[PARTS][CH];
	__shared__ float s_w[KV_SPLITS], s_ref[KV_WAVES], s_sum[KV_WAVES];
	const int kv_head = blockIdx.x % a.kv_heads, mine = blockIdx.x / a.kv_heads, s = blockIdx.y;
	__shared__ int s_from[2];
	const kv_seq sq = kv_sequence(a, s);
	if (mine >= sq.n * G)
		return;
	if (shares) { /* the first share that the sequence is in, and their count */
		const kv_line line = kv_line_of(a, window);
		const int share = kv_share(line.all, shares);
		if ((int)threadIdx.x == s) {
			s_from[0] = line.start / share;
			s_from[1] = (line.start + line.tiles - 1) / share + 1 - s_from[0];
		}
		__syncthreads();
	}
	const int rt = mine / KV_ROWS, i = mine / G, base = sq.len - sq.n;
	const int i0 = rt * KV_ROWS / G, i1 = (min(rt * KV_ROWS + KV_ROWS, sq.n * G) - 1) / G;
	const int first = window ? max(0, base + i0 + 1 - window) : 0, last = max(base + i1 + 1, 0);
	const int tiles = (last + KV_TILE - 1) / KV_TILE - first / KV_TILE;
	const int n = shares ? s_from[1] : min(splits, max(1, (tiles + chunk - 1) / chunk));
	const size_t piece = shares ? (size_t)kv_head * (shares + a.nseq) + s_from[0] + s
				    : ((size_t)(s * row_tiles + rt) * a.kv_heads + kv_head) * splits;
	const float *p = ws + piece * nrows * (D + 4) + mine % KV_ROWS * (D + 4);
	const int c = threadIdx.x % CH, part = threadIdx.x / CH;
	const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
	const size_t step = nrows * (D + 4);

	/* every piece's reference and sum, then its weight */
	constexpr int PER = KV_SPLITS / KV_NT;
	float r[PER], l[PER], ref = -__builtin_inff(), sum = 0.0f;
#pragma unroll
	for (int u = 0; u < PER; u++) {
		const int at = threadIdx.x + u * KV_NT;
		r[u] = at < n ? p[at * step + D] : -__builtin_inff();
		l[u] = at < n ? p[at * step + D + 1] : 0.0f;
		ref = fmaxf(ref, r[u]);
	}
	for (int o = WAVE / 2; o > 0; o >>= 1)
		ref = fmaxf(ref, __shfl_xor(ref, o, WAVE));
	if (lane == 0)
		s_ref[wave] = ref;
	__syncthreads();
#pragma unroll
	for (int u = 0; u < KV_WAVES; u++)
		ref = fmaxf(ref, s_ref[u]);
#pragma unroll
	for (int u = 0; u < PER; u++) {
		const float f = weight(r[u], ref);
		s_w[threadIdx.x + u * KV_NT] = f;
		sum += l[u] * f;
	}
	for (int o = WAVE / 2; o > 0; o >>= 1)
		sum += __shfl_xor(sum, o, WAVE);
	if (lane == 0)
		s_sum[wave] = sum;
	__syncthreads();
	floatx4 y = (floatx4)0.0f;
#pragma unroll 8
	for (int u = part; u < n; u += PARTS)
		y += *(const floatx4 *)(p + u * step + 4 * c) * s_w[u];
	s_y[part][c] = y;
	__syncthreads();
	if (part)
		return;
#pragma unroll
	for (int u = 1; u < PARTS; u++)
		y += s_y[u][c];
	sum = s_sum[0];
#pragma unroll
	for (int u = 1; u < KV_WAVES; u++)
		sum += s_sum[u];
	kv_vec<TY, 4> z;
#pragma unroll
	for (int u = 0; u < 4; u++)
		z.v[u] = T::put(base + i >= 0 ? y[u] / sum : 0.0f);
	*(kv_vec<TY, 4> *)(out + (size_t)(sq.row + i) * out_stride + (size_t)(kv_head * G + mine - i * G) * D +
			   4 * c) = z;
}

/*
 * Many query rows: tiles of 32 of them on v_mfma_f32_32x32x16_f16, which needs half
 * the instructions and whose lanes hold 16 scores of one query row: the row's
 * statistics cost half as much a score, and a tile's codes are made f16 once for 32
 * rows.  The layout serves it as it is: lane l (c = l / 32) takes row l % 32 of the
 * keys, 8-channel parts c and 2 + c of a group in two steps; the scores of cached
 * rows 8 i + 4 c + (0 .. 3), i < 4, come out in it, of which i = 0 and 2 are the rows
 * of value words c, i = 1 and 3 those of words 2 + c.  Row 16 e + m of channel tile
 * 2 b + u is channel 64 b + 16 (2 e + u) + m, so that a lane's words lie together.
 *
 * A workgroup's four waves share 32 query rows and deal the cache's tiles among
 * them, and the row tiles that see most come first: even the last workgroups are
 * short.
 *
 * 8192 bf16 rows of 32 heads on 8 of 128: 905 to 945 us, 600 TFLOP/s of the formula's
 * operations (in tiles of 16 rows 1.5 ms); 347 instructions on the vector unit's side for
 * 32 x 32 scores, 19 of them matrix instructions of 32 cycles.  2048 fp32 rows of 16 heads
 * on as many cached: 54.6 us (in two parts, 620 TFLOP/s).  Waves with 32 rows each that share a tile's f16 codes
 * through LDS took 8 to 12 % longer: the barrier a tile keeps matrix and VALU work of
 * the two waves of a SIMD from overlapping.
 */
#define KV_WIDE 32

template <int D> struct kv_keys32 {
	typedef kv_tile<D> L;
	u32 w[2][L::G];       /* part c and 2 + c of row lane % 32 */
	u32x4 d[4][L::G / 2]; /* scales of rows 8 i + 4 c + j */
	u32 own[L::G / 2];    /* of row lane % 32 */
	__device__ inline void load(const uint8_t *tile, int lane)
	{
		typedef uint32_t words __attribute__((ext_vector_type(L::P)));
		const int c = lane / 32, r = lane % 32;
#pragma unroll
		for (int h = 0; h < 2; h++)
#pragma unroll
			for (int g = 0; g < L::G; g += L::P) {
				const words x = ((const words *)tile)[(r / 16 * (L::G / L::P) + g / L::P) * 64 +
								      16 * (2 * h + c) + r % 16];
#pragma unroll
				for (int u = 0; u < L::P; u++)
					w[h][g + u] = x[u];
			}
#pragma unroll
		for (int i = 0; i < 4; i++)
#pragma unroll
			for (int u = 0; u < L::G / 2; u++)
				d[i][u] = ((const u32x4 *)(tile + L::K_SCALES))[(8 * i + 4 * c) * L::G / 8 + u];
#pragma unroll
		for (int u = 0; u < L::G / 2; u++)
			own[u] = ((const u32 *)(tile + L::K_SCALES))[r * L::G / 2 + u];
	}
	/* the row's scales, twice: the operand that k_kv_attn_wide's surplus is
	 * multiplied with */
	__device__ inline half8_t scales8() const
	{
		u32 w[4] = {};
#pragma unroll
		for (int u = 0; u < L::G / 2; u++) {
			w[u] = w[2 + u] = own[u];
		}
		return as_half8(w[0], w[1], w[2], w[3]);
	}
	__device__ inline float scale(int i, int j, int g) const
	{
		return (float)__builtin_bit_cast(half8_t, d[i][(j * L::G + g) / 8])[(j * L::G + g) % 8];
	}
};

template <int D> struct kv_values32 {
	u32x2 w[D / 64][2]; /* parts c and 2 + c of rows 16 e + m of channel tiles 2 b and 2 b + 1 */
	u32x2 d[4];         /* scales of rows 8 i + 4 c + j */
	__device__ inline void load(const uint8_t *tile, int lane)
	{
		typedef kv_tile<D> L;
		const int c = lane / 32, e = lane / 16 % 2, m = lane % 16;
#pragma unroll
		for (int b = 0; b < D / 64; b++)
#pragma unroll
			for (int h = 0; h < 2; h++)
				w[b][h] = ((const u32x2 *)(tile + L::V_CODES))[(64 * b + 16 * (2 * h + c) + m) * 2 + e];
#pragma unroll
		for (int i = 0; i < 4; i++)
			d[i] = ((const u32x2 *)(tile + L::V_SCALES))[2 * i + c];
	}
};

/* (heads of 64 in fp32 fit four waves a SIMD: 4096 rows of 32 heads on 8 201 us; with
 * one register too many for that 209) */
template <int D, int TY>
__global__ __launch_bounds__(KV_NT) __attribute__((amdgpu_waves_per_eu(D == 64 && TY == HIP_KV_F32 ? 4 : 2)))
void k_kv_attn_wide(kv_args a, const typename kv_type<TY>::t *q, size_t q_stride, int G,
		    typename kv_type<TY>::t *out, size_t out_stride, float scale, int window, int row_tiles)
{
	typedef kv_type<TY> T;
	typedef kv_tile<D> L;
	constexpr int QP = TY == HIP_KV_F32 ? 2 : 1, PP = TY == HIP_KV_BF16 ? 1 : 2;
	constexpr int CT = D / 32;
	/* the queries' parts, [part][group][step][lane], then the waves' outputs */
	__shared__ union {
		half8_t q[QP][L::G][2][WAVE];
		float o[KV_WAVES][KV_WIDE][D + 4];
	} sh;
	__shared__ float s_ref[KV_WAVES][KV_WIDE], s_sum[KV_WAVES][KV_WIDE];
	__shared__ int s_row[KV_WIDE], s_head[KV_WIDE];

	const int lane = threadIdx.x % WAVE, part = lane / 32;
	const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
	const int kv_head = blockIdx.x % a.kv_heads, s = blockIdx.z;
	const int rt = row_tiles - 1 - (int)(blockIdx.x / a.kv_heads);
	const kv_seq sq = kv_sequence(a, s);
	if (rt * KV_WIDE >= sq.n * G)
		return;
	const kv_span r = kv_rows_of<KV_WIDE>(sq, rt, G, kv_head, window, lane);
	const int t0 = r.first / KV_TILE, t1 = (max(r.last, 0) + KV_TILE - 1) / KV_TILE;
	float rs;
	half8_t surplus = (half8_t)(_Float16)0.0f;
	{
		/* the lane's parts 2 h + c of each group, of which the wave puts its own
		 * share of the groups into LDS */
		kv_vec<TY, 8> w[2 * L::G];
#pragma unroll
		for (int u = 0; u < 2 * L::G; u++)
			w[u] = *(const kv_vec<TY, 8> *)(q + (size_t)r.row * q_stride + (size_t)r.head * D +
							32 * (u / 2) + 8 * (u % 2 * 2 + part));
		float top = 0.0f;
#pragma unroll
		for (int u = 0; u < 2 * L::G; u++)
#pragma unroll
			for (int j = 0; j < 8; j++)
				top = fmaxf(top, fabsf(T::get(w[u].v[j])));
		const kv_factor f = kv_query_factor<TY>(half_max(top), scale, kv_form<TY>::STEP);
		rs = f.score;
#pragma unroll
		for (int u = 0; u < L::G; u++) {
			float sum = 0.0f;
#pragma unroll
			for (int h = 0; h < 2; h++) {
				half8_t z[QP];
				sum += kv_split8<QP, TY>(w[2 * u + h], f.query, z);
#pragma unroll
				for (int p = 0; p < QP; p++)
					if (u % KV_WAVES == wave)
						sh.q[p][u][h][lane] = z[p];
			}
			/* in two f16 parts (of at most 1 and 2^-12) */
			sum = -8.0f * kv_form<TY>::STEP * half_sum(sum);
			if (!kv_form<TY>::EVEN && part == 0) {
				surplus[u] = (_Float16)sum;
				surplus[4 + u] = rest(sum, surplus[u]);
			}
		}
	}
	if (threadIdx.x < KV_WIDE) {
		s_row[threadIdx.x] = r.valid ? r.row : -1;
		s_head[threadIdx.x] = r.hi > r.lo ? r.head : ~r.head;
	}

	const int shift = a.page_shift - 5;
	const int32_t *table = a.table + s * a.table_stride;
	const int n = a.pages ? (t1 - t0 - wave + KV_WAVES - 1) / KV_WAVES : 0;
	int page = -1;
	bool lost = false;
	const auto tile_of = [&](int i) -> const uint8_t * {
		const int t = t0 + wave + i * KV_WAVES;
		if (i % WAVE == 0) {
			const int tl = t + lane * KV_WAVES;
			page = tl < t1 ? table[tl >> shift] : -1;
		}
		const int id = __builtin_amdgcn_readlane(page, i % WAVE);
		lost = (u32)id >= (u32)a.pages;
		const size_t at = lost ? 0 : ((((size_t)id * a.kv_heads + kv_head) << shift) + (t & ((1 << shift) - 1)));
		return a.pool + at * L::BYTES;
	};
	kv_keys32<D> k;
	kv_values32<D> v;
	if (n > 0) {
		const uint8_t *tile = tile_of(0);
		k.load(tile, lane);
		v.load(tile, lane);
	} else if (!a.pages && t1 > t0 && lane == 0) {
		kv_error(a, HIP_KV_ERR_PAGE);
	}
	/* For bf16 outputs the values' surplus of 8 leaves at the end, as 8 times the
	 * sum of the (rounded) probabilities times scales: it outweighs the output by
	 * up to 3 times the root of the rows that matter, which fp32 sums have to
	 * spare over bf16's 8 bits: over 131072 rows whose scales have one sign and
	 * whose values cancel, outputs are 1.7e-3 off, by their rounding. */
	constexpr bool LATE = TY == HIP_KV_BF16;
	floatx16 o[CT], late = (floatx16)0.0f;
#pragma unroll
	for (int c = 0; c < CT; c++)
		o[c] = (floatx16)0.0f;
	kv_soft soft = {-__builtin_inff(), 0.0f};
	__syncthreads();

	for (int i = 0; i < n; i++) {
		const int t = t0 + wave + i * KV_WAVES;
		const bool hidden = lost;
		const uint8_t *next = tile_of(min(i + 1, n - 1));
		half2_t dv[8];
		kv_halves<16> pp[PP];
		floatx16 x = (floatx16)0.0f;
		if (!kv_form<TY>::EVEN)
			x = __builtin_amdgcn_mfma_f32_32x32x16_f16(k.scales8(), surplus, x, 0, 0, 0);
#pragma unroll
		for (int g = 0; g < L::G; g++) {
			floatx16 acc = (floatx16)0.0f;
#pragma unroll
			for (int h = 0; h < 2; h++) {
				const half8_t kf = kv_form<TY>::EVEN ? kv_word8<TY>(k.w[h][g]) : kv_word(k.w[h][g]);
#pragma unroll
				for (int p = 0; p < QP; p++)
					acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, sh.q[p][g][h][lane], acc, 0, 0, 0);
			}
#pragma unroll
			for (int j = 0; j < 16; j++)
				x[j] = fmaf(k.scale(j / 4, j % 4, g), acc[j], x[j]);
		}
		/* the scales are used up before their registers are loaded again */
		asm volatile("" : "+v"(x) : : "memory");
		k.load(next, lane);
#pragma unroll
		for (int j = 0; j < 4; j++) {
			const u32x2 w = v.d[j];
			const u32 lo = w.x, hi = w.y; /* (bit_cast takes no element) */
			dv[2 * j] = __builtin_bit_cast(half2_t, lo);
			dv[2 * j + 1] = __builtin_bit_cast(half2_t, hi);
		}
		if (hidden || t * KV_TILE < r.inner0 || (t + 1) * KV_TILE > r.inner1) {
			const int lo = hidden ? 0x7fffffff : r.lo;
#pragma unroll
			for (int j = 0; j < 16; j++) {
				const int at = t * KV_TILE + 8 * (j / 4) + 4 * part + j % 4;
				const bool hide = at < lo || at >= r.hi;
				x[j] = hide ? -__builtin_inff() : x[j];
				dv[j / 2][j % 2] = hide ? (_Float16)0.0f : dv[j / 2][j % 2];
			}
			if (hidden && lane == 0)
				kv_error(a, HIP_KV_ERR_PAGE);
		}
		half8_t pf[2][PP];
		kv_softmax<16, 2, PP, TY>(soft, (const float *)&x, dv, rs, 0.0f, pp, [&](float back) {
			late *= back;
#pragma unroll
			for (int c = 0; c < CT; c++)
				o[c] *= back;
		});
		/* rows 8 i + .. are in step i % 2, codes 4 (i / 2) .. of the words */
#pragma unroll
		for (int p = 0; p < PP; p++) {
			pf[0][p] = __builtin_shufflevector(pp[p], pp[p], 0, 1, 2, 3, 8, 9, 10, 11);
			pf[1][p] = __builtin_shufflevector(pp[p], pp[p], 4, 5, 6, 7, 12, 13, 14, 15);
		}
#pragma unroll
		for (int c = 0; c < CT; c++)
#pragma unroll
			for (int h = 0; h < 2; h++) {
				const u32 w = v.w[c / 2][h][c % 2];
				const half8_t vf = LATE ? kv_word(w) : kv_word8<TY>(w);
#pragma unroll
				for (int p = 0; p < PP; p++)
					o[c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pf[h][p], o[c], 0, 0, 0);
			}
		if (LATE)
#pragma unroll
			for (int h = 0; h < 2; h++)
				late = __builtin_amdgcn_mfma_f32_32x32x16_f16(kv_surplus8(), pf[h][0], late, 0, 0, 0);
		v.load(next, lane);
	}
	if (LATE)
#pragma unroll
		for (int c = 0; c < CT; c++)
			o[c] -= late;

	/* the waves' results: to one reference, then added in wave order */
	const float sum = kv_form<TY>::STEP * half_sum(soft.sum);
	if (part == 0)
		s_ref[wave][lane] = soft.ref;
	__syncthreads();
	float ref = s_ref[0][lane % 32];
#pragma unroll
	for (int w = 1; w < KV_WAVES; w++)
		ref = fmaxf(ref, s_ref[w][lane % 32]);
	const float factor = weight(soft.ref, ref);
	if (part == 0)
		s_sum[wave][lane] = sum * factor;
#pragma unroll
	for (int c = 0; c < CT; c++)
#pragma unroll
		for (int i = 0; i < 4; i++) {
			floatx4 y;
#pragma unroll
			for (int j = 0; j < 4; j++)
				y[j] = o[c][4 * i + j] * factor;
			*(floatx4 *)&sh.o[wave][lane % 32][64 * (c / 2) + 16 * (i / 2 * 2 + c % 2) +
							    8 * (i % 2) + 4 * part] = y;
		}
	__syncthreads();
	for (int at = threadIdx.x; at < KV_WIDE * D / 4; at += KV_NT) {
		const int i = at / (D / 4), c = at % (D / 4) * 4, row = s_row[i], head = s_head[i];
		if (row < 0)
			break;
		float den = s_sum[0][i];
		floatx4 y = *(const floatx4 *)&sh.o[0][i][c];
#pragma unroll
		for (int w = 1; w < KV_WAVES; w++) {
			den += s_sum[w][i];
			y += *(const floatx4 *)&sh.o[w][i][c];
		}
		kv_vec<TY, 4> z;
#pragma unroll
		for (int u = 0; u < 4; u++)
			z.v[u] = T::put(head >= 0 ? y[u] / den : 0.0f);
		*(kv_vec<TY, 4> *)(out + row * out_stride + (size_t)(head < 0 ? ~head : head) * D + c) = z;
	}
}

/*
 * Along the cache.  A workgroup of KV_MANY waves takes a row tile's whole cache where
 * that beats pieces, which need a second launch to add them up: up to 32 tiles, 72
 * where there are 128 workgroups and 128 where there are 512, which fill the chip by
 * themselves.  32 heads on 8 of 128 in fp32, whole and in pieces: 1 sequence x 2048 rows
 * 15.1 and 11.2 us; 8 x 1100 rows 11.0 and 11.4, 16 x 11.3 and 13.8, 32 x 11.9 and 17.7;
 * 8 x 2300 rows 17.8 and 13.8, 16 x 17.9 and 17.4, 32 x 18.6 and 24.5, 64 x 37.9 and 48;
 * 32 x 4000 rows 33.5 and 36.6, 48 x 60.6 and 54.7, 64 x 58.5 and 66.8.  Other caches are cut into pieces for
 * workgroups of four waves, as many as the chip holds twice over for heads of 64 and
 * 128 (131072 rows: 64 pieces a kv head 35.4 us, 128 pieces 36.3), and of several
 * sequences into pieces of at most KV_CHUNK tiles, so that different lengths fill the
 * chip evenly (64 sequences of 340 to 16384 rows: pieces of 16 tiles 107 us, 32 tiles
 * 100, 64 tiles 111, 128 tiles 140).
 *
 * Of many sequences, where the longest that may come would be 4096 pieces in all and
 * more, most of which find nothing to do (launching one costs its XCD 90 cycles), the
 * caches are one line in equal shares, as many as the chip holds: the same 64 88 us
 * instead of 97.5, 96 110 instead of 130, 64 of 8190 rows each (bf16) 115.5 instead of
 * 118.6.  Finding a share's sequences costs 2 us a launch, so that fewer lose where their
 * lengths are equal (8190 rows: 48 93 instead of 91, 32 64.5 instead of 62.7, 16 38.8
 * instead of 34.6; one of 131072 rows 39.5 instead of 35.4), though 32 and 48 of 340 to
 * 16384 rows would gain (50 instead of 55, 67 instead of 76): they begin at 512 workgroups,
 * where both gain.
 */
#define KV_CHUNK 32
#define KV_MANY 8

extern "C" void kv_attn_plan(const kv_args *a, int head_len, int heads, int window, kv_plan *p)
{
	const int G = heads / a->kv_heads;
	const long all = ((long)a->max_len + KV_TILE - 1) / KV_TILE;
	long tiles = all; /* of the cache that one tile of query rows sees, at most */
	if (window && (long)window + KV_ROWS < a->max_len)
		tiles = ((long)window + KV_ROWS + KV_TILE - 2) / KV_TILE + 1;
	tiles = tiles < all ? tiles : all;
	const long rows = (long)a->max_rows * G;
	p->row_tiles = (int)((rows + KV_ROWS - 1) / KV_ROWS);
	p->rows = (int)(rows < KV_ROWS ? rows : KV_ROWS);
	/* slots: 64 sequences x 4000 rows, 32 fp32 heads on 8: 52.8 us with four, 61.4 with
	 * two, 66.3 without; 64 heads on 8 in 16 bits: 46.0 with two, 56.8 without */
	p->slots = rows <= 4 && head_len > 64 ? 4 : rows <= 8 ? 2 : 1;
	const size_t wgs = (size_t)a->nseq * a->kv_heads * p->row_tiles;
	p->shares = 0;
	/* tiles of 32 rows (heads of 256 have no registers for them) where they fill the
	 * chip: 8 x 64 rows on 2048, 32 heads on 8: 35.5 us, in tiles of 16 41.8; 512
	 * workgroups only on longer caches: 512 rows of 16 heads alone 13.2 and 12.3, 4 x 64
	 * rows of 32 heads of 64 on 4096 44.2 and 49.5 */
	p->wide = head_len < 256 && rows >= 2 * KV_WIDE && (wgs >= 1024 || (wgs >= 512 && all >= 32));
	if (p->wide) {
		p->row_tiles = (int)((rows + KV_WIDE - 1) / KV_WIDE);
		p->splits = 1;
		p->ws = 0;
		return;
	}
	const size_t room = head_len == 64 ? 1024 : head_len == 128 ? 512 : 256;
	const long by_room = wgs < room ? (long)(room / wgs) : 1;
	const long whole = head_len < 256 && p->row_tiles == 1 ? wgs < 128 ? 32 : wgs < 512 ? 72 : 128 : 0;
	p->waves = whole && tiles <= whole ? KV_MANY : KV_WAVES; /* (no tiles at all: max_len 0) */
	const size_t pieces = (size_t)a->nseq * a->kv_heads * ((all + KV_CHUNK - 1) / KV_CHUNK);
	if (p->row_tiles == 1 && all > whole && a->nseq <= KV_SEQS && wgs >= 512 && pieces >= 4096 &&
	    (size_t)a->nseq * all < (size_t)1 << 30) {
		const int chip = head_len == 256 ? 512 : 1024, shares = a->kv_heads < chip ? chip / a->kv_heads : 1;
		/* (never less than shorter bounds need) */
		const size_t slots = (size_t)a->kv_heads * (shares + a->nseq);
		p->ws = (slots > 4096 ? slots : 4096) * p->rows * (head_len + 4) * sizeof(float);
		p->shares = tiles > whole ? shares : 0;
		p->splits = p->shares ? shares : 1;
		p->chunk = (int)tiles;
		return;
	}
	long chunk = (tiles + by_room - 1) / by_room;
	if (wgs >= room / 8 && chunk > KV_CHUNK && p->row_tiles == 1)
		chunk = KV_CHUNK;
	if (chunk < (tiles + KV_SPLITS - 1) / KV_SPLITS)
		chunk = (tiles + KV_SPLITS - 1) / KV_SPLITS;
	if (p->waves > KV_WAVES)
		chunk = tiles;
	/* many rows cost the merge more than short pieces save: 256 rows of 16 heads alone
	 * 16.8 us in two pieces of 4 tiles, 8.0 in one of 8 */
	const long least = p->row_tiles > 4 ? 2 * KV_WAVES : KV_WAVES;
	p->chunk = (int)(chunk < least ? least : chunk);
	p->splits = (int)((tiles + p->chunk - 1) / p->chunk);
	p->splits = p->splits < 1 ? 1 : p->splits;
	/* without regard to the window, so that one workspace serves any: pieces by
	 * room, or of KV_CHUNK tiles, and none below KV_WAVES */
	const long by_chunk = (all + KV_CHUNK - 1) / KV_CHUNK, few = (all + least - 1) / least;
	long most = p->row_tiles == 1 && by_chunk > by_room ? by_chunk : by_room;
	most = most < few ? most : few;
	most = most < KV_SPLITS ? most : KV_SPLITS;
	if (all <= whole)
		most = 1;
	p->ws = most > 1 ? wgs * most * p->rows * (head_len + 4) * sizeof(float) : 0;
}

extern "C" int kv_launch_attn(const kv_args *a, int head_len, int type, const void *q,
			      size_t q_stride, int heads, void *out, size_t out_stride, float scale,
			      int window, void *ws, const kv_plan *p, void *stream)
{
	const int G = heads / a->kv_heads;
	const size_t tiles = (size_t)a->kv_heads * p->row_tiles, all = (size_t)heads * a->max_rows;
	const bool merge = !p->wide && (p->splits > 1 || p->shares);
	if (!kv_launchable(tiles, KV_MANY * WAVE) || (merge && !kv_launchable(all, KV_NT)))
		return (int)hipErrorInvalidConfiguration;
	const dim3 grid((unsigned)tiles, (unsigned)p->splits, (unsigned)a->nseq);
	const dim3 rows((unsigned)all, (unsigned)a->nseq);
	KV_DISPATCH_HEAD(head_len, D, KV_DISPATCH_TYPE(type, TY, {
		typedef kv_type<TY>::t t;
		constexpr int WIDE = D < 256 ? D : 128; /* heads of 256 have no registers for it */
		if (p->wide) {
			k_kv_attn_wide<WIDE, TY><<<grid, KV_NT, 0, (hipStream_t)stream>>>(
				*a, (const t *)q, q_stride, G, (t *)out, out_stride, scale, window,
				p->row_tiles);
			return (int)hipGetLastError();
		}
		/* (heads of 256 have no room for KV_MANY waves, of 64 no four groups) */
		constexpr int MANY = D < 256 ? KV_MANY : KV_WAVES, FOUR = D > 64 ? 4 : 2;
		const auto launch = [&](auto kernel, int waves) { /* as many as it is made for */
			kernel<<<dim3(grid.x, grid.y, p->shares ? 1 : grid.z), waves * WAVE, 0, (hipStream_t)stream>>>(
				*a, (const t *)q, q_stride, G, (t *)out, out_stride, scale, window, (float *)ws,
				p->row_tiles, p->chunk, p->rows);
		};
		if (p->shares)
			launch(p->slots == 4 ? k_kv_attn<D, TY, KV_WAVES, FOUR, true> :
			       p->slots == 2 ? k_kv_attn<D, TY, KV_WAVES, 2, true> : k_kv_attn<D, TY, KV_WAVES, 1, true>, KV_WAVES);
		else if (p->waves == KV_MANY)
			launch(p->slots == 4 ? k_kv_attn<D, TY, MANY, FOUR, false> :
			       p->slots == 2 ? k_kv_attn<D, TY, MANY, 2, false> : k_kv_attn<D, TY, MANY, 1, false>, MANY);
		else
			launch(p->slots == 4 ? k_kv_attn<D, TY, KV_WAVES, FOUR, false> :
			       p->slots == 2 ? k_kv_attn<D, TY, KV_WAVES, 2, false> : k_kv_attn<D, TY, KV_WAVES, 1, false>, KV_WAVES);
		if (merge)
			k_kv_merge<D, TY><<<rows, KV_NT, 0, (hipStream_t)stream>>>(
				*a, G, (t *)out, out_stride, window, (const float *)ws, p->row_tiles,
				p->chunk, p->splits, p->rows, p->shares);
	}))
	return (int)hipGetLastError();
}
