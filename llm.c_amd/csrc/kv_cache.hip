/*
 * kv_cache.hip - rotary positions, and rows of keys and values into and out of
 * the paged 4-bit cache (include/hip_kv.h has the formulas and the layout).
 */
#include "kv_device.h"

#define KV_NT 256

/*
 * cos and sin, times mag, of the angle pos * freq in 64 bits.  The quarter turns n
 * nearest to the angle go off it in three steps, pi / 2 as a sum of three doubles
 * (Cody and Waite's reduction), each step one rounding; what is left, up to pi / 4 in size, goes through the Taylor
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

/* A row's (cos, sin) in LDS, by pair: one place is left free after eight, so that
 * lanes that each read eight or four in a row do not meet in the same banks */
__host__ __device__ static inline int kv_slot(int pair)
{
	return pair + (pair >> 3);
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
	const double b = (double)other * t.y;
	return (float)fma((double)own, t.x, first ? -b : b);
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
				const double2 t = turns[kv_slot((c0 + u) / 2)];
				const float a = y[u], b = y[u + 1];
				y[u] = kv_turned(a, b, true, t);
				y[u + 1] = kv_turned(b, a, false, t);
			}
		} else if (half % N == 0) {
			const bool first = c0 < half;
#pragma unroll
			for (int u = 0; u < N; u++)
				y[u] = kv_turned(y[u], T::get(other.v[u]), first, turns[kv_slot((first ? c0 : c0 - half) + u)]);
		} else {
			for (int u = 0; u < N && c0 + u < rot; u++) {
				const int c = c0 + u;
				const bool first = c < half;
				y[u] = kv_turned(y[u], T::get(x[first ? c + half : c - half]), first,
						 turns[kv_slot(first ? c : c - half)]);
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
 *
 * Bound by HBM: 8192 rows of 32 bf16 heads of 128 (134 MB) in 32 us, 4.2 TB/s where a
 * large copy has 5.1 (48 us with angles and 4-byte accesses head by head); 16 rows of
 * a step in 3.5 us.
 */
#define KV_ROPE_ROWS 8 /* rows of a workgroup, at most */

template <int TY, bool VEC>
__global__ __launch_bounds__(KV_NT) void k_kv_rope(
	const typename kv_type<TY>::t *x, size_t x_stride, typename kv_type<TY>::t *out,
	size_t out_stride, int rows, int heads, int head_len, hip_rope R, const int32_t *pos, int per,
	int heads_per)
{
	typedef kv_type<TY> T;
	extern __shared__ double2 turns[]; /* [rows][kv_slot(rot / 2)] */
	const int half = (int)R.rot / 2, slots = kv_slot(half), r0 = blockIdx.x * per, n = min(per, rows - r0);
	const bool pairs = R.layout == HIP_ROPE_PAIRS;
	x += (size_t)blockIdx.y * heads_per * head_len;
	out += (size_t)blockIdx.y * heads_per * head_len;
	heads = min(heads_per, heads - (int)blockIdx.y * heads_per);
	for (int at = threadIdx.x; at < n * half; at += KV_NT)
		turns[at / half * slots + kv_slot(at % half)] = kv_turn(R, pos[r0 + at / half], at % half);
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
			const double2 *t = turns + r * slots;
			vec a = *(const vec *)xr;
			if (pairs) {
#pragma unroll
				for (int u = 0; u < N; u += 2) {
					if (c + u >= 2 * half)
						continue;
					const float y1 = T::get(a.v[u]), y2 = T::get(a.v[u + 1]);
					const double2 z = t[kv_slot((c + u) / 2)];
					a.v[u] = T::put(kv_turned(y1, y2, true, z));
					a.v[u + 1] = T::put(kv_turned(y2, y1, false, z));
				}
			} else if (c < half) {
				vec b = *(const vec *)(xr + half);
#pragma unroll
				for (int u = 0; u < N; u++) {
					const float y1 = T::get(a.v[u]), y2 = T::get(b.v[u]);
					a.v[u] = T::put(kv_turned(y1, y2, true, t[kv_slot(c + u)]));
					b.v[u] = T::put(kv_turned(y2, y1, false, t[kv_slot(c + u)]));
				}
				*(vec *)(yr + half) = b;
			}
			*(vec *)yr = a;
		}
		return;
	}
	const int own = half + (head_len - 2 * half), all = n * heads * own;
	for (int at = threadIdx.x; at < all; at += KV_NT) {
		const int i = at % own, h = at / own % heads, r = at / own / heads;
		const typename T::t *xr = x + (size_t)(r0 + r) * x_stride + h * head_len;
		typename T::t *yr = out + (size_t)(r0 + r) * out_stride + h * head_len;
		if (i >= half) { /* a channel that passes */
			yr[i + half] = xr[i + half];
			continue;
		}
		const int c1 = pairs ? 2 * i : i, c2 = pairs ? 2 * i + 1 : i + half;
		const float a = T::get(xr[c1]), b = T::get(xr[c2]);
		yr[c1] = T::put(kv_turned(a, b, true, turns[r * slots + kv_slot(i)]));
		yr[c2] = T::put(kv_turned(b, a, false, turns[r * slots + kv_slot(i)]));
	}
}

/* ---------------------------------------------------------------------- */
/* storing rows                                                           */
/* ---------------------------------------------------------------------- */

/* A value's bits turned left by one order values by size, the negative one of two
 * equal last, and NaN behind all */
__device__ static inline u32 kv_key(float v)
{
	return kv_rotr(__builtin_bit_cast(u32, v), 31);
}

/* the largest key of the LANES lanes around this one: within 16 lanes by mirrored
 * halves, which after the first steps hold equal values */
template <int LANES> __device__ static inline u32 kv_most(u32 v)
{
	if (LANES > 1)
		v = max(v, (u32)__builtin_amdgcn_mov_dpp((int)v, 0xb1, 0xf, 0xf, true)); /* lane ^ 1 */
	if (LANES > 2)
		v = max(v, (u32)__builtin_amdgcn_mov_dpp((int)v, 0x4e, 0xf, 0xf, true)); /* lane ^ 2 */
	if (LANES > 4)
		v = max(v, (u32)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xf, 0xf, true)); /* 7 - lane of 8 */
	if (LANES > 8)
		v = max(v, (u32)__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xf, 0xf, true)); /* 15 - lane of 16 */
	if (LANES > 16) {
		const auto t = __builtin_amdgcn_permlane16_swap(v, v, false, false);
		v = max((u32)t[0], (u32)t[1]);
	}
	if (LANES > 32) {
		const auto t = __builtin_amdgcn_permlane32_swap(v, v, false, false);
		v = max((u32)t[0], (u32)t[1]);
	}
	return v;
}

/*
 * The scale of a group of values that LANES lanes hold N each of, and the lane's
 * codes floor(y / d + 8.5) within 0 .. 15, exactly.  In fp32, y * (1 / d) + 8.5 is
 * within 2^-19 of what it stands for (2^-24 of 1 / d, times 8.1 at most, and half a
 * step of 16); where a value lies that near to a border the lanes look again, by the
 * sign of y - (q - 8.5) d, which one fma has (the product holds 16 bits).
 */
template <int LANES, int N> __device__ static inline _Float16 kv_encode(const float *y, u32 *codes)
{
	u32 key = kv_key(y[0]);
#pragma unroll
	for (int u = 1; u < N; u++)
		key = max(key, kv_key(y[u]));
	const float m = __builtin_bit_cast(float, kv_rotr(kv_most<LANES>(key), 1)) * -0.125f;
	const _Float16 d = (_Float16)(fabsf(m) > 65504.0f ? copysignf(65504.0f, m) : m);
	const float df = (float)d, inv = df == 0.0f ? 0.0f : 1.0f / df;
	float q[N], off = 0.0f;
#pragma unroll
	for (int u = 0; u < N; u++) {
		const float t = fmaf(y[u], inv, 8.5f);
		q[u] = floorf(t);
		off = fmaxf(off, fabsf(t - q[u] - 0.5f));
	}
	if (__ballot(off > 0.5f - 0x1p-18f)) {
		const float w = fabsf(df);
#pragma unroll
		for (int u = 0; u < N; u++) {
			const float v = df < 0.0f ? -y[u] : y[u];
			const float below = fmaf(8.5f - q[u], w, v), above = fmaf(7.5f - q[u], w, v);
			q[u] += (above >= 0.0f ? 1.0f : 0.0f) - (below < 0.0f ? 1.0f : 0.0f);
		}
		/* (a scale of 0 stands for 0: code 8) */
#pragma unroll
		for (int u = 0; u < N; u++)
			q[u] = w > 0.0f ? q[u] : 8.0f;
	}
#pragma unroll
	for (int u = 0; u < N; u++)
		codes[u] = (u32)__builtin_amdgcn_fmed3f(q[u], 0.0f, 15.0f);
	return d;
}

/*
 * One workgroup: the call's rows among the eight of one tile of one sequence that
 * share value words (4 part + (0 .. 3) of each half), for `per` kv heads and as large
 * a share of the q heads: few rows and many heads, since each workgroup works out the
 * angles of its rows, into LDS.  Then a wave takes a row and as many heads as it has
 * lanes for (16 bytes of a head row a lane) at a time, keys and values or queries.
 * Keys meet their group's scale, values their row's, over a few lanes.  The value codes
 * go to LDS: the words are put together from there, and a word that has other rows'
 * codes too is read first and keeps them.
 *
 * 8192 fp32 rows of 8 kv and 32 q heads of 128 (345 MB) take 86 us, 4.0 TB/s: HBM.
 * 7971 bf16 rows of 16 and 16 heads in five sequences (148 MB, 29 us of a large copy)
 * take 59: VALU work, about 40 instructions for a key or value and 16 for a query's, of
 * which full issue would take 35 us, beside waits for loads, of which a workgroup's first
 * are behind its sequence's length and page.  With 32 rows and two heads a workgroup: 88
 * and 62.5 us.
 */
#define KV_APPEND_NT 512
#define KV_PART 8 /* rows of a workgroup, at most */

template <int D, int TY>
__global__ __launch_bounds__(KV_APPEND_NT) void k_kv_append(
	kv_args a, hip_rope R, const typename kv_type<TY>::t *k, const typename kv_type<TY>::t *v,
	size_t kv_stride, const int32_t *pos, const typename kv_type<TY>::t *q, size_t q_stride,
	int heads, typename kv_type<TY>::t *q_out, size_t q_out_stride, int per, int tiles, int parts)
{
	typedef kv_type<TY> T;
	typedef kv_tile<D> L;
	constexpr int N = kv_wide<TY>::N, HL = D / N; /* lanes of a head row */
	constexpr int HP = WAVE / HL;                 /* heads of a wave's step */
	constexpr int GL = 32 / N;                    /* lanes of a key group */
	typedef typename kv_wide<TY>::vec vec;
	extern __shared__ double2 turns[]; /* [rows][kv_slot(rot / 2)], then the codes [per][rows][D] */
	const int half = (int)R.rot / 2, slots = kv_slot(half);
	const int most = parts > 1 ? KV_PART : 1;
	uint8_t *codes = (uint8_t *)(turns + most * slots);

	const int groups = (a.kv_heads + per - 1) / per;
	const int hg = blockIdx.x % groups, unit = blockIdx.x / groups % (tiles * parts);
	const int s = blockIdx.x / groups / (tiles * parts);
	const kv_seq sq = kv_sequence(a, s);
	const int base = sq.len - sq.n, p0 = max(0, base), t = p0 / KV_TILE + unit / parts;
	if (t >= (sq.len + KV_TILE - 1) / KV_TILE) /* (t * KV_TILE may pass 31 bits) */
		return;
	/* the part (a single row's own), and its rows i0 .. i0 + n - 1 in their order: row
	 * 16 (i / 4) + 4 part + i % 4 of the tile */
	const int part = parts > 1 ? unit % parts : p0 % 16 / 4;
	const auto row_of = [&](int i) { return i / 4 * 16 + 4 * part + i % 4; };
	const auto below = [&](int r) { /* rows of the part before row r of the tile */
		return min(4, max(0, r - 4 * part)) + min(4, max(0, r - 16 - 4 * part));
	};
	const int i0 = below(p0 - t * KV_TILE), n = below(min(sq.len - t * KV_TILE, KV_TILE)) - i0;
	if (n <= 0)
		return;
	const int row0 = sq.row + t * KV_TILE - base; /* + r: row r of the tile among the call's */
	const int h0 = hg * per, h1 = min(h0 + per, a.kv_heads);
	const int q0 = q ? (int)((long)heads * h0 / a.kv_heads) : 0;
	const int q1 = q ? (int)((long)heads * h1 / a.kv_heads) : 0;
	const bool pairs = R.layout == HIP_ROPE_PAIRS;
	/* the page: one for the tile */
	const int shift = a.page_shift - 5, id = a.table[s * a.table_stride + (t >> shift)];
	uint8_t *const page = (u32)id < (u32)a.pages
		? a.pool + ((((size_t)id * a.kv_heads) << shift) + (t & ((1 << shift) - 1))) * L::BYTES : NULL;
	const size_t head_bytes = (size_t)L::BYTES << shift;
	if (!page && threadIdx.x == 0)
		kv_error(a, HIP_KV_ERR_PAGE);

	const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), lane = threadIdx.x % WAVE;
	const int sub = lane / HL, c0 = lane % HL * N;
	const int ks = page ? (h1 - h0 + HP - 1) / HP : 0, steps = ks + (q1 - q0 + HP - 1) / HP;
	constexpr int NW = KV_APPEND_NT / WAVE;
	/* a step's vectors, loaded a step ahead */
	struct item {
		kv_turn_in<TY> in;
		vec val;
		const typename T::t *x;
		int i, h; /* row of the part, head; h < 0: query head ~h */
	};
	const auto fetch = [&](int at) {
		item z;
		z.i = at / steps;
		const int step = at % steps;
		const size_t row = row0 + row_of(i0 + z.i);
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
	for (int at = threadIdx.x; at < n * half; at += KV_APPEND_NT) {
		const int i = at / half, r = row_of(i0 + i);
		turns[i * slots + kv_slot(at % half)] = kv_turn(R, pos ? pos[row0 + r] : t * KV_TILE + r, at % half);
	}
	__syncthreads();
	for (int at = wave; at < n * steps; at += NW) {
		const item z = next;
		if (at + NW < n * steps)
			next = fetch(at + NW);
		const int i = z.i;
		float y[N];
		z.in.turn(z.x, c0, 2 * half, pairs, turns + i * slots, y);
		if (at % steps >= ks) {
			vec o;
#pragma unroll
			for (int u = 0; u < N; u++)
				o.v[u] = T::put(y[u]);
			__builtin_amdgcn_wave_barrier(); /* in place: the lanes' loads come first */
			*(vec *)(q_out + (size_t)(row0 + row_of(i0 + i)) * q_out_stride + (size_t)~z.h * D + c0) = o;
			continue;
		}
		uint8_t *const tile = page + z.h * head_bytes;
		const int r = row_of(i0 + i);
		u32 z4[N], w = 0;
		_Float16 d = kv_encode<GL, N>(y, z4);
#pragma unroll
		for (int u = 0; u < N; u++)
			w |= z4[u] << kv_bit(u);
		if (N == 8)
			w |= z4[N - 1] >> 2; /* code 7 wraps */
		if (N == 4) { /* codes 0 .. 3 and, of the next lane, 4 .. 7 */
			if (c0 % 8)
				w = kv_rotr(w, 24);
			w |= (u32)__builtin_amdgcn_mov_dpp((int)w, 0xb1, 0xf, 0xf, true);
		}
		if (c0 % 8 == 0)
			((u32 *)tile)[L::k_word(r, c0)] = w;
		if (c0 % 32 == 0)
			((_Float16 *)(tile + L::K_SCALES))[r * L::G + c0 / 32] = d;

#pragma unroll
		for (int u = 0; u < N; u++)
			y[u] = T::get(z.val.v[u]);
		d = kv_encode<HL, N>(y, z4);
		u32 *to = (u32 *)&codes[((z.h - h0) * most + i) * D + c0];
#pragma unroll
		for (int u = 0; u < N; u += 4)
			to[u / 4] = z4[u] | z4[u + 1] << 8 | z4[u + 2] << 16 | z4[u + 3] << 24;
		if (c0 == 0)
			((_Float16 *)(tile + L::V_SCALES))[r] = d;
	}
	__syncthreads();
	if (!page)
		return;

	/* four words that lie together: channels 64 b + m, + 16, + 32, + 48 */
	u32 mine = 0;
	for (int j = 0; j < n; j++)
		mine |= kv_rotr(15, 32 - kv_bit(i0 + j));
	for (int at = threadIdx.x; at < (h1 - h0) * D / 4; at += KV_APPEND_NT) {
		const int h = at / (D / 4), b = at % (D / 4) / 16, c = 64 * b + at % 16;
		u32 w[4] = {};
#pragma unroll
		for (int j = 0; j < KV_PART; j++) {
			if (j < i0 || j >= i0 + n)
				continue;
#pragma unroll
			for (int u = 0; u < 4; u++)
				w[u] |= kv_rotr(codes[(h * most + j - i0) * D + c + 16 * u], 32 - kv_bit(j));
		}
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
 * channels of a row at a time.  8192 fp32 rows of 8 heads of 128 (76 MB): 17 us,
 * 4.4 TB/s. */
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
	if (t >= (sq.len + KV_TILE - 1) / KV_TILE)
		return;
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
	return (int)(((long)n + 2 * KV_TILE - 2) / KV_TILE);
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
	if (!kv_launchable((rows + per - 1) / per, KV_NT))
		return (int)hipErrorInvalidConfiguration;
	const dim3 grid((unsigned)((rows + per - 1) / per), (unsigned)((heads + heads_per - 1) / heads_per));
	const size_t lds = per * kv_slot((int)R->rot / 2) * sizeof(double2);
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
	const int tiles = kv_tiles_of(a->max_rows), parts = a->max_rows > 1 ? 4 : 1;
	/* all kv heads a workgroup (32 KB of codes at most) where the rows alone
	 * are two workgroups a CU; else fewer, down to one */
	const int most = parts > 1 ? KV_PART : 1;
	int per = 1;
	const int top = 32768 / (KV_PART * head_len);
	while (per < top && per < a->kv_heads &&
	       (size_t)a->nseq * tiles * parts * ((a->kv_heads + 2 * per - 1) / (2 * per)) >= 512)
		per *= 2;
	per = per < a->kv_heads ? per : a->kv_heads;
	const size_t grid = (size_t)a->nseq * tiles * parts * ((a->kv_heads + per - 1) / per);
	if (!kv_launchable(grid, KV_APPEND_NT))
		return (int)hipErrorInvalidConfiguration;
	const size_t lds = (size_t)most * ((R ? kv_slot((int)R->rot / 2) * sizeof(double2) : 0) + (size_t)per * head_len);
	KV_DISPATCH_HEAD(head_len, D, KV_DISPATCH_TYPE(type, TY, {
		typedef kv_type<TY>::t t;
		k_kv_append<D, TY><<<dim3((unsigned)grid), KV_APPEND_NT, lds, (hipStream_t)stream>>>(
			*a, R ? *R : none, (const t *)k, (const t *)v, kv_stride, pos, (const t *)q,
			q_stride, heads, (t *)q_out, q_out_stride, per, tiles, parts);
	}))
	return (int)hipGetLastError();
}

extern "C" int kv_launch_read(const kv_args *a, int head_len, int type, void *k, void *v,
			      size_t stride, void *stream)
{
	const int tiles = kv_tiles_of(a->max_rows);
	const size_t grid = (size_t)a->nseq * tiles * a->kv_heads;
	if (!kv_launchable(grid, KV_NT))
		return (int)hipErrorInvalidConfiguration;
	KV_DISPATCH_HEAD(head_len, D, KV_DISPATCH_TYPE(type, TY, {
		typedef kv_type<TY>::t t;
		k_kv_read<D, TY><<<dim3((unsigned)grid), KV_NT, 0, (hipStream_t)stream>>>(
			*a, (t *)k, (t *)v, stride, tiles);
	}))
	return (int)hipGetLastError();
}
