/*
 * kv_cache.hip - rotary positions, and rows of keys and values into and out of
 * the paged 4-bit cache (include/hip_kv.h has the formulas and the layout).
 */
#include "kv_device.h"

#define KV_NT 256

/*
 * cos and sin, times mag, of the angle pos * freq in 64 bits.  The quarter turns n
 * nearest to the angle go off it in three steps, pi / 2 as a sum of three doubles,
 * each step one rounding; what is left, up to pi / 4 in size, goes through the Taylor
 * series of both functions, whose first terms left out are below 2^-54 of 1; n mod 4
 * says which is which.  Within 2^-52 of the functions' values, at a fifth of the
 * instructions of a function for any argument (which takes the angles past 2^31).
 */
__device__ static inline double2 kv_turn(const hip_rope &R, int pos, int i)
{
	const double a = (double)pos * R.freq[i];
	double c, s;
	if (fabs(a) < 2147483648.0) {
		const double n = rint(a * 0.63661977236758134308);
		double y = fma(n, -0x1.921fb544p+0, a);
		y = fma(n, -0x1.0b4611a6p-34, y);
		y = fma(n, -0x1.3198a2e037073p-69, y);
		const double z = y * y;
		double p = -1.0 / 1307674368000.0, q = 1.0 / 20922789888000.0;
		p = fma(p, z, 1.0 / 6227020800.0);
		q = fma(q, z, -1.0 / 87178291200.0);
		p = fma(p, z, -1.0 / 39916800.0);
		q = fma(q, z, 1.0 / 479001600.0);
		p = fma(p, z, 1.0 / 362880.0);
		q = fma(q, z, -1.0 / 3628800.0);
		p = fma(p, z, -1.0 / 5040.0);
		q = fma(q, z, 1.0 / 40320.0);
		p = fma(p, z, 1.0 / 120.0);
		q = fma(q, z, -1.0 / 720.0);
		p = fma(p, z, -1.0 / 6.0);
		q = fma(q, z, 1.0 / 24.0);
		const double sn = fma(y * z, p, y), cs = fma(z, fma(q, z, -0.5), 1.0);
		const int k = (int)n & 3;
		c = k & 1 ? sn : cs;
		s = k & 1 ? cs : sn;
		c = k == 1 || k == 2 ? -c : c;
		s = k >= 2 ? -s : s;
	} else {
		sincos(a, &s, &c);
	}
	return make_double2(c * R.mag, s * R.mag);
}

/* 16 bytes of values */
template <int TY> struct kv_wide {
	static constexpr int N = 16 / sizeof(typename kv_type<TY>::t);
	typedef kv_vec<TY, N> vec;
};

/* value u (channel c) of a vector whose turned partners are at x[c + other]:
 * cs and sn belong to channel c's pair */
__device__ static inline float kv_turned(float own, float other, bool first, double2 t)
{
	const double a = (double)own * t.x, b = (double)other * t.y;
	return (float)(first ? a - b : a + b);
}

/* The vector x[c0 ..] of a head row with what its turn needs: in HALVES, where half
 * the rotated channels are whole vectors, the vector of the other values */
template <int TY> struct kv_turn_in {
	typename kv_wide<TY>::vec own, other;
	__device__ inline void load(const typename kv_type<TY>::t *x, int c0, int rot, bool pairs)
	{
		typedef typename kv_wide<TY>::vec vec;
		own = *(const vec *)(x + c0);
		if (!pairs && rot / 2 % kv_wide<TY>::N == 0 && c0 < rot)
			other = *(const vec *)(x + (c0 < rot / 2 ? c0 + rot / 2 : c0 - rot / 2));
	}
	/* its channels below rot turned by `turns`, the row's (cos, sin) by pair; x is
	 * read again where the others are not a vector */
	__device__ inline void turn(const typename kv_type<TY>::t *x, int c0, int rot, bool pairs,
				    const double2 *turns, float *y) const
	{
		typedef kv_type<TY> T;
		constexpr int N = kv_wide<TY>::N;
		const int half = rot / 2;
#pragma unroll
		for (int u = 0; u < N; u++)
			y[u] = T::get(own.v[u]);
		if (c0 >= rot)
			return;
		if (pairs) {
#pragma unroll
			for (int u = 0; u < N; u += 2) {
				if (c0 + u >= rot)
					continue;
				const double2 t = turns[(c0 + u) / 2];
				const float a = y[u], b = y[u + 1];
				y[u] = kv_turned(a, b, true, t);
				y[u + 1] = kv_turned(b, a, false, t);
			}
		} else if (half % N == 0) {
			const bool first = c0 < half;
#pragma unroll
			for (int u = 0; u < N; u++)
				y[u] = kv_turned(y[u], T::get(other.v[u]), first, turns[(first ? c0 : c0 - half) + u]);
		} else {
			for (int u = 0; u < N && c0 + u < rot; u++) {
				const int c = c0 + u;
				const bool first = c < half;
				y[u] = kv_turned(y[u], T::get(x[first ? c + half : c - half]), first,
						 turns[first ? c : c - half]);
			}
		}
	}
};

/* ---------------------------------------------------------------------- */
/* rotation                                                               */
/* ---------------------------------------------------------------------- */

/*
 * A workgroup takes `per` rows: their angles once, into LDS, then its heads.
 * VEC: rows, strides and channels in whole vectors of 16 bytes; else value by value.
 * A thread computes both values of a pair before it stores either, so that it may
 * work in place: with VEC and HALVES it takes a vector and its partner.
 */
#define KV_ROPE_ROWS 8 /* rows of a workgroup, at most */

template <int TY, bool VEC>
__global__ __launch_bounds__(KV_NT) void k_kv_rope(
	const typename kv_type<TY>::t *x, size_t x_stride, typename kv_type<TY>::t *out,
	size_t out_stride, int rows, int heads, int head_len, hip_rope R, const int32_t *pos, int per,
	int heads_per)
{
	typedef kv_type<TY> T;
	extern __shared__ double2 turns[]; /* [rows][rot / 2] */
	const int half = (int)R.rot / 2, r0 = blockIdx.x * per, n = min(per, rows - r0);
	const bool pairs = R.layout == HIP_ROPE_PAIRS;
	x += (size_t)blockIdx.y * heads_per * head_len;
	out += (size_t)blockIdx.y * heads_per * head_len;
	heads = min(heads_per, heads - (int)blockIdx.y * heads_per);
	for (int at = threadIdx.x; at < n * half; at += KV_NT)
		turns[at] = kv_turn(R, pos[r0 + at / half], at % half);
	__syncthreads();
	if (VEC) {
		constexpr int N = kv_wide<TY>::N;
		typedef typename kv_wide<TY>::vec vec;
		/* vectors of a head that a thread takes by itself or with its partner */
		const int mine = (pairs ? head_len : head_len - half) / N, all = n * heads * mine;
#pragma unroll 4
		for (int at = threadIdx.x; at < all; at += KV_NT) {
			const int v = at % mine, h = at / mine % heads, r = at / mine / heads;
			/* HALVES: the first half with the second, then what passes */
			const int c = v * N, c0 = pairs || c < half ? c : c + half;
			const typename T::t *xr = x + (size_t)(r0 + r) * x_stride + h * head_len + c0;
			typename T::t *yr = out + (size_t)(r0 + r) * out_stride + h * head_len + c0;
			const double2 *t = turns + r * half;
			vec a = *(const vec *)xr;
			if (pairs) {
#pragma unroll
				for (int u = 0; u < N; u += 2) {
					if (c + u >= 2 * half)
						continue;
					const float y1 = T::get(a.v[u]), y2 = T::get(a.v[u + 1]);
					const double2 z = t[(c + u) / 2];
					a.v[u] = T::put(kv_turned(y1, y2, true, z));
					a.v[u + 1] = T::put(kv_turned(y2, y1, false, z));
				}
			} else if (c < half) {
				vec b = *(const vec *)(xr + half);
#pragma unroll
				for (int u = 0; u < N; u++) {
					const float y1 = T::get(a.v[u]), y2 = T::get(b.v[u]);
					a.v[u] = T::put(kv_turned(y1, y2, true, t[c + u]));
					b.v[u] = T::put(kv_turned(y2, y1, false, t[c + u]));
				}
				*(vec *)(yr + half) = b;
			}
			*(vec *)yr = a;
		}
		return;
	}
	const int slots = half + (head_len - 2 * half), all = n * heads * slots;
	for (int at = threadIdx.x; at < all; at += KV_NT) {
		const int i = at % slots, h = at / slots % heads, r = at / slots / heads;
		const typename T::t *xr = x + (size_t)(r0 + r) * x_stride + h * head_len;
		typename T::t *yr = out + (size_t)(r0 + r) * out_stride + h * head_len;
		if (i >= half) { /* a channel that passes */
			yr[i + half] = xr[i + half];
			continue;
		}
		const int c1 = pairs ? 2 * i : i, c2 = pairs ? 2 * i + 1 : i + half;
		const float a = T::get(xr[c1]), b = T::get(xr[c2]);
		yr[c1] = T::put(kv_turned(a, b, true, turns[r * half + i]));
		yr[c2] = T::put(kv_turned(b, a, false, turns[r * half + i]));
	}
}

/* ---------------------------------------------------------------------- */
/* storing rows                                                           */
/* ---------------------------------------------------------------------- */

/* the scale of a group whose smallest and largest values are lo and hi */
__device__ static inline _Float16 kv_scale(float lo, float hi)
{
	const float m = hi > -lo ? hi : lo;
	return (_Float16)fminf(fmaxf(m * -0.125f, -65504.0f), 65504.0f);
}

/* floor(x / d + 8.5) within 0 .. 15, exactly: the quotient's estimate is
 * put right by the sign of x - (q - 8.5) d, which one fma has (the product
 * holds 16 bits).  inv is 1 / |d|. */
__device__ static inline u32 kv_code(float x, float d, float inv)
{
	const float y = d < 0.0f ? -x : x, w = fabsf(d);
	float q = floorf(fminf(fmaxf(y * inv, -8.5f), 8.5f) + 8.5f);
	q = fmaf(8.5f - q, w, y) < 0.0f ? q - 1.0f : fmaf(7.5f - q, w, y) >= 0.0f ? q + 1.0f : q;
	return w == 0.0f ? 8 : (u32)fminf(fmaxf(q, 0.0f), 15.0f);
}

/* the smallest (the largest) of the LANES lanes around this one: within 16 lanes
 * by mirrored halves, which after the first steps hold equal values */
template <int CTRL> __device__ static inline float kv_dpp(float v)
{
	return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}

template <int LANES, class Fn> __device__ static inline float kv_over(float v, Fn fn)
{
	if (LANES > 1)
		v = fn(v, kv_dpp<0xb1>(v)); /* lane ^ 1 */
	if (LANES > 2)
		v = fn(v, kv_dpp<0x4e>(v)); /* lane ^ 2 */
	if (LANES > 4)
		v = fn(v, kv_dpp<0x141>(v)); /* 7 - lane of 8 */
	if (LANES > 8)
		v = fn(v, kv_dpp<0x140>(v)); /* 15 - lane of 16 */
	if (LANES > 16)
		v = fn(v, __shfl_xor(v, 16, WAVE));
	if (LANES > 32)
		v = fn(v, __shfl_xor(v, 32, WAVE));
	return v;
}

/* the scale of the group of values that LANES lanes hold N each of; NaN if one of
 * them is */
template <int LANES, int N> __device__ static inline _Float16 kv_group(const float *y)
{
	float lo = y[0], hi = y[0], any = 0.0f;
#pragma unroll
	for (int u = 0; u < N; u++) {
		lo = fminf(lo, y[u]);
		hi = fmaxf(hi, y[u]);
		any = y[u] != y[u] ? y[u] : any;
	}
	lo = kv_over<LANES>(lo, [](float a, float b) { return fminf(a, b); });
	hi = kv_over<LANES>(hi, [](float a, float b) { return fmaxf(a, b); });
	any = kv_over<LANES>(any, [](float a, float b) { return a + b; });
	return any == any ? kv_scale(lo, hi) : (_Float16)__builtin_nanf("");
}

/*
 * One workgroup: the call's rows in one tile of one sequence, for `per` kv heads
 * and as large a share of the q heads.  The rows' angles go into LDS once; then a
 * wave takes a row and as many heads as it has lanes for (16 bytes of a head row a
 * lane) at a time, keys and values or queries.  Keys meet their group's scale, values
 * their row's, over a few lanes.  The value codes go to LDS, since one word holds
 * eight rows' codes of a channel: the words are put together from there, and a word
 * that has other rows' codes too is read first and keeps them.
 */
#define KV_APPEND_NT 512

template <int D, int TY>
__global__ __launch_bounds__(KV_APPEND_NT) void k_kv_append(
	kv_args a, hip_rope R, const typename kv_type<TY>::t *k, const typename kv_type<TY>::t *v,
	size_t kv_stride, const int32_t *pos, const typename kv_type<TY>::t *q, size_t q_stride,
	int heads, typename kv_type<TY>::t *q_out, size_t q_out_stride, int per, int tiles, int most)
{
	typedef kv_type<TY> T;
	typedef kv_tile<D> L;
	constexpr int N = kv_wide<TY>::N, HL = D / N; /* lanes of a head row */
	constexpr int HP = WAVE / HL;                 /* heads of a wave's step */
	constexpr int GL = 32 / N;                    /* lanes of a key group */
	typedef typename kv_wide<TY>::vec vec;
	extern __shared__ double2 turns[]; /* [most][rot / 2], then the codes [per][most][D] */
	const int half = (int)R.rot / 2;
	uint8_t *codes = (uint8_t *)(turns + most * half);

	const int groups = (a.kv_heads + per - 1) / per;
	const int hg = blockIdx.x % groups, tb = blockIdx.x / groups % tiles;
	const int s = blockIdx.x / groups / tiles;
	const kv_seq sq = kv_sequence(a, s);
	const int base = sq.len - sq.n, p0 = max(0, base), t = p0 / KV_TILE + tb;
	const int lo = max(p0, t * KV_TILE), hi = min(sq.len, (t + 1) * KV_TILE);
	if (lo >= hi)
		return;
	const int n = hi - lo, r0 = lo % KV_TILE, row0 = sq.row + lo - base;
	const int h0 = hg * per, h1 = min(h0 + per, a.kv_heads);
	const int q0 = q ? (int)((long)heads * h0 / a.kv_heads) : 0;
	const int q1 = q ? (int)((long)heads * h1 / a.kv_heads) : 0;
	const bool pairs = R.layout == HIP_ROPE_PAIRS;
	for (int at = threadIdx.x; at < n * half; at += KV_APPEND_NT) {
		const int r = at / half;
		turns[at] = kv_turn(R, pos ? pos[row0 + r] : lo + r, at % half);
	}
	/* the page: one for the tile */
	const int shift = a.page_shift - 5, id = a.table[s * a.table_stride + (t >> shift)];
	uint8_t *const page = (u32)id < (u32)a.pages
		? a.pool + ((((size_t)id * a.kv_heads) << shift) + (t & ((1 << shift) - 1))) * L::BYTES : NULL;
	const size_t head_bytes = (size_t)L::BYTES << shift;
	if (!page && threadIdx.x == 0)
		kv_error(a, HIP_KV_ERR_PAGE);
	__syncthreads();

	const int wave = threadIdx.x / WAVE, lane = threadIdx.x % WAVE;
	const int sub = lane / HL, c0 = lane % HL * N;
	const int ks = page ? (h1 - h0 + HP - 1) / HP : 0, steps = ks + (q1 - q0 + HP - 1) / HP;
	constexpr int NW = KV_APPEND_NT / WAVE;
	/* a step's vectors, loaded a step ahead */
	struct item {
		kv_turn_in<TY> in;
		vec val;
		const typename T::t *x;
		int i, h; /* row of the tile, head; h < 0: query head ~h */
	};
	const auto fetch = [&](int at) {
		item z;
		z.i = at / steps;
		const int step = at % steps;
		const size_t row = row0 + z.i;
		if (step >= ks) {
			const int h = min(q0 + (step - ks) * HP + sub, q1 - 1); /* (the last head again) */
			z.h = ~h;
			z.x = q + row * q_stride + (size_t)h * D;
		} else {
			z.h = min(h0 + step * HP + sub, h1 - 1);
			z.x = k + row * kv_stride + (size_t)z.h * D;
			z.val = *(const vec *)(v + row * kv_stride + (size_t)z.h * D + c0);
		}
		z.in.load(z.x, c0, 2 * half, pairs);
		return z;
	};
	item next;
	if (wave < n * steps)
		next = fetch(wave);
	for (int at = wave; at < n * steps; at += NW) {
		const item z = next;
		if (at + NW < n * steps)
			next = fetch(at + NW);
		const int i = z.i;
		float y[N];
		z.in.turn(z.x, c0, 2 * half, pairs, turns + i * half, y);
		if (at % steps >= ks) {
			vec o;
#pragma unroll
			for (int u = 0; u < N; u++)
				o.v[u] = T::put(y[u]);
			__builtin_amdgcn_wave_barrier(); /* in place: the lanes' loads come first */
			*(vec *)(q_out + (size_t)(row0 + i) * q_out_stride + (size_t)~z.h * D + c0) = o;
			continue;
		}
		uint8_t *const tile = page + z.h * head_bytes;
		const int r = r0 + i;
		_Float16 d = kv_group<GL, N>(y);
		float df = (float)d, inv = df == 0.0f ? 0.0f : 1.0f / fabsf(df);
		u32 w = 0;
#pragma unroll
		for (int u = 0; u < N; u++)
			w |= kv_rotr(kv_code(y[u], df, inv), 32 - kv_bit((c0 + u) % 8));
		if (N == 4)
			w |= (u32)__builtin_amdgcn_mov_dpp((int)w, 0xb1, 0xf, 0xf, true);
		if (c0 % 8 == 0)
			((u32 *)tile)[L::k_word(r, c0)] = w;
		if (c0 % 32 == 0)
			((_Float16 *)(tile + L::K_SCALES))[r * L::G + c0 / 32] = d;

#pragma unroll
		for (int u = 0; u < N; u++)
			y[u] = T::get(z.val.v[u]);
		d = kv_group<HL, N>(y);
		df = (float)d;
		inv = df == 0.0f ? 0.0f : 1.0f / fabsf(df);
		uint8_t b[N];
#pragma unroll
		for (int u = 0; u < N; u++)
			b[u] = (uint8_t)kv_code(y[u], df, inv);
		__builtin_memcpy(__builtin_assume_aligned(&codes[((z.h - h0) * most + i) * D + c0], N), b, N);
		if (c0 == 0)
			((_Float16 *)(tile + L::V_SCALES))[r] = d;
	}
	__syncthreads();
	if (!page)
		return;

	/* four words that lie together: channels 64 b + m, + 16, + 32, + 48 */
	for (int at = threadIdx.x; at < (h1 - h0) * D; at += KV_APPEND_NT) {
		const int h = at / D, b = at % D / 64, part = at % 64 / 16, c = 64 * b + at % 16;
		u32 w[4] = {}, mine = 0;
#pragma unroll
		for (int j = 0; j < 8; j++) {
			const int r = j / 4 * 16 + part * 4 + j % 4 - r0;
			if (r < 0 || r >= n)
				continue;
			mine |= kv_rotr(15, 32 - kv_bit(j));
#pragma unroll
			for (int u = 0; u < 4; u++)
				w[u] |= kv_rotr(codes[(h * most + r) * D + c + 16 * u], 32 - kv_bit(j));
		}
		if (!mine)
			continue;
		u32x4 *to = (u32x4 *)(page + (h0 + h) * head_bytes + L::V_CODES) + L::v_word(part * 4, c) / 4;
		u32x4 old = {w[0], w[1], w[2], w[3]};
		if (~mine)
			old |= *to & ~mine;
		*to = old;
	}
}

/* ---------------------------------------------------------------------- */
/* reading rows                                                           */
/* ---------------------------------------------------------------------- */

/* One workgroup: the batch's rows in one tile of one sequence and kv head.  The
 * value words, of eight rows each, are taken apart into LDS; then a thread takes 8
 * channels of a row at a time. */
template <int D, int TY>
__global__ __launch_bounds__(KV_NT) void k_kv_read(kv_args a, typename kv_type<TY>::t *k,
						    typename kv_type<TY>::t *v, size_t stride,
						    int tiles)
{
	typedef kv_type<TY> T;
	typedef kv_tile<D> L;
	__shared__ uint8_t codes[KV_TILE][D];
	const int h = blockIdx.x % a.kv_heads, tb = blockIdx.x / a.kv_heads % tiles;
	const int s = blockIdx.x / a.kv_heads / tiles;
	const kv_seq sq = kv_sequence(a, s);
	const int base = sq.len - sq.n, p0 = max(0, base), t = p0 / KV_TILE + tb;
	const int lo = max(p0, t * KV_TILE), hi = min(sq.len, (t + 1) * KV_TILE);
	if (lo >= hi)
		return;
	const uint8_t *tile = kv_tile_at<D>(a, s, h, t);
	if (!tile) {
		if (threadIdx.x == 0)
			kv_error(a, HIP_KV_ERR_PAGE);
		return;
	}
	for (int at = threadIdx.x; at < D; at += KV_NT) { /* four words that lie together */
		const int b = at / 64, part = at % 64 / 16, c = 64 * b + at % 16;
		const u32x4 w = ((const u32x4 *)(tile + L::V_CODES))[L::v_word(part * 4, c) / 4];
#pragma unroll
		for (int u = 0; u < 4; u++) {
			const u32 x = w[u];
#pragma unroll
			for (int j = 0; j < 8; j++)
				codes[j / 4 * 16 + part * 4 + j % 4][c + 16 * u] = (uint8_t)(kv_rotr(x, kv_bit(j)) & 15);
		}
	}
	__syncthreads();
	for (int at = threadIdx.x; at < (hi - lo) * (D / 8); at += KV_NT) {
		const int c = at % (D / 8) * 8, p = lo + at / (D / 8), r = p % KV_TILE;
		const size_t to = (size_t)(sq.row + p - base) * stride + (size_t)h * D + c;
		const u32 kw = ((const u32 *)tile)[L::k_word(r, c)];
		const float kd = (float)((const _Float16 *)(tile + L::K_SCALES))[r * L::G + c / 32];
		const float vd = (float)((const _Float16 *)(tile + L::V_SCALES))[r];
		uint8_t z[8];
		__builtin_memcpy(z, __builtin_assume_aligned(&codes[r][c], 8), 8);
		kv_vec<TY, 8> ko, vo;
#pragma unroll
		for (int j = 0; j < 8; j++) {
			ko.v[j] = T::put((float)((int)(kv_rotr(kw, kv_bit(j)) & 15) - 8) * kd);
			vo.v[j] = T::put((float)((int)z[j] - 8) * vd);
		}
		*(kv_vec<TY, 8> *)(k + to) = ko;
		*(kv_vec<TY, 8> *)(v + to) = vo;
	}
}

/* ---------------------------------------------------------------------- */
/* launchers                                                              */
/* ---------------------------------------------------------------------- */

/* tiles that n consecutive rows of a sequence can touch, at most */
static int kv_tiles_of(int n)
{
	return (n + 2 * KV_TILE - 2) / KV_TILE;
}

extern "C" int kv_launch_rope(int type, const void *x, size_t x_stride, void *out,
			      size_t out_stride, size_t rows, int heads, int head_len,
			      const hip_rope *R, const int32_t *pos, void *stream)
{
	/* a workgroup computes its rows' angles once for its heads: as many of both
	 * as leave two workgroups a CU */
	int per = KV_ROPE_ROWS, heads_per = heads;
	while (per > 1 && rows / per < 512)
		per /= 2;
	while (heads_per > 4 && rows * ((heads + heads_per - 1) / heads_per) < 512)
		heads_per = (heads_per + 1) / 2;
	const dim3 grid((unsigned)((rows + per - 1) / per), (unsigned)((heads + heads_per - 1) / heads_per));
	const size_t lds = per * (R->rot / 2) * sizeof(double2);
	KV_DISPATCH_TYPE(type, TY, {
		typedef kv_type<TY>::t t;
		const size_t n = kv_wide<TY>::N;
		const bool vec = !((uintptr_t)x % 16 || (uintptr_t)out % 16 || x_stride % n || out_stride % n ||
				   head_len % n || (R->layout == HIP_ROPE_HALVES && R->rot / 2 % n));
		if (vec)
			k_kv_rope<TY, true><<<grid, KV_NT, lds, (hipStream_t)stream>>>(
				(const t *)x, x_stride, (t *)out, out_stride, (int)rows, heads, head_len, *R, pos, per,
				heads_per);
		else
			k_kv_rope<TY, false><<<grid, KV_NT, lds, (hipStream_t)stream>>>(
				(const t *)x, x_stride, (t *)out, out_stride, (int)rows, heads, head_len, *R, pos, per,
				heads_per);
	})
	return (int)hipGetLastError();
}

extern "C" int kv_launch_append(const kv_args *a, int head_len, int type, const hip_rope *R,
				const void *k, const void *v, size_t kv_stride,
				const int32_t *pos, const void *q, size_t q_stride, int heads,
				void *q_out, size_t q_out_stride, void *stream)
{
	const hip_rope none = {0, HIP_ROPE_PAIRS, NULL, 1.0};
	const int tiles = kv_tiles_of(a->max_rows), most = a->max_rows < KV_TILE ? a->max_rows : KV_TILE;
	/* all kv heads a workgroup (32 KB of codes at most) where the tiles alone
	 * are two a CU; else fewer, down to one */
	int per = 1;
	const int top = 32768 / (KV_TILE * head_len);
	while (per < top && per < a->kv_heads && (size_t)a->nseq * tiles * a->kv_heads / (2 * per) >= 512)
		per *= 2;
	per = per < a->kv_heads ? per : a->kv_heads;
	const size_t grid = (size_t)a->nseq * tiles * ((a->kv_heads + per - 1) / per);
	const size_t lds = (size_t)most * ((R ? R->rot / 2 * sizeof(double2) : 0) + (size_t)per * head_len);
	KV_DISPATCH_HEAD(head_len, D, KV_DISPATCH_TYPE(type, TY, {
		typedef kv_type<TY>::t t;
		k_kv_append<D, TY><<<dim3((unsigned)grid), KV_APPEND_NT, lds, (hipStream_t)stream>>>(
			*a, R ? *R : none, (const t *)k, (const t *)v, kv_stride, pos, (const t *)q,
			q_stride, heads, (t *)q_out, q_out_stride, per, tiles, most);
	}))
	return (int)hipGetLastError();
}

extern "C" int kv_launch_read(const kv_args *a, int head_len, int type, void *k, void *v,
			      size_t stride, void *stream)
{
	const int tiles = kv_tiles_of(a->max_rows);
	const size_t grid = (size_t)a->nseq * tiles * a->kv_heads;
	KV_DISPATCH_HEAD(head_len, D, KV_DISPATCH_TYPE(type, TY, {
		typedef kv_type<TY>::t t;
		k_kv_read<D, TY><<<dim3((unsigned)grid), KV_NT, 0, (hipStream_t)stream>>>(
			*a, (t *)k, (t *)v, stride, tiles);
	}))
	return (int)hipGetLastError();
}
