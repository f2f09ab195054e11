/*
 * kv_cache.hip - rotary positions, and rows of keys and values into and out of
 * the paged 4-bit cache (include/hip_kv.h has the formulas and the layout).
 */
#include "kv_device.h"

#define KV_NT 256

/* cos and sin, times mag, of position p for pair i */
__device__ static inline void kv_turn(const hip_rope &R, int p, int i, double *c, double *s)
{
	sincos((double)p * R.freq[i], s, c);
	*c *= R.mag;
	*s *= R.mag;
}

/* ---------------------------------------------------------------------- */
/* rotation                                                               */
/* ---------------------------------------------------------------------- */

/*
 * A workgroup takes rows of its grid, its threads the pairs of a row (and the
 * channels that pass): each computes its angle once for all heads.
 */
template <int TY>
__global__ __launch_bounds__(KV_NT) void k_kv_rope(
	const typename kv_type<TY>::t *x, size_t x_stride, typename kv_type<TY>::t *out,
	size_t out_stride, int rows, int heads, int head_len, hip_rope R, const int32_t *pos)
{
	typedef kv_type<TY> T;
	const int half = (int)R.rot / 2, slots = half + (head_len - (int)R.rot);
	for (long at = (long)blockIdx.x * KV_NT + threadIdx.x; at < (long)rows * slots;
	     at += (long)gridDim.x * KV_NT) {
		const int r = (int)(at / slots), i = (int)(at % slots);
		const typename T::t *xr = x + r * x_stride;
		typename T::t *yr = out + r * out_stride;
		if (i >= half) { /* a channel that passes */
			const int c = i + half;
			for (int h = 0; h < heads; h++)
				yr[h * head_len + c] = xr[h * head_len + c];
			continue;
		}
		double c, s;
		kv_turn(R, pos[r], i, &c, &s);
		const int c1 = R.layout == HIP_ROPE_PAIRS ? 2 * i : i;
		const int c2 = R.layout == HIP_ROPE_PAIRS ? 2 * i + 1 : i + half;
		for (int h = 0; h < heads; h++) {
			const double a = (double)T::get(xr[h * head_len + c1]);
			const double b = (double)T::get(xr[h * head_len + c2]);
			yr[h * head_len + c1] = T::put((float)(a * c - b * s));
			yr[h * head_len + c2] = T::put((float)(b * c + a * s));
		}
	}
}

/* ---------------------------------------------------------------------- */
/* storing rows                                                           */
/* ---------------------------------------------------------------------- */

/* the scale of a group whose smallest and largest values are lo and hi (NaN
 * if one of them is: see kv_group) */
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
	if (fmaf(8.5f - q, w, y) < 0.0f)
		q -= 1.0f;
	else if (fmaf(7.5f - q, w, y) >= 0.0f)
		q += 1.0f;
	return w == 0.0f ? 8 : (u32)fminf(fmaxf(q, 0.0f), 15.0f);
}

/* VPL channels of a head row from channel c0 on, turned where R.rot says */
template <int TY, int VPL>
__device__ static inline void kv_turned(const typename kv_type<TY>::t *x, int c0, const hip_rope &R,
					const double *cs, const double *sn, float *y)
{
	typedef kv_type<TY> T;
	const int rot = (int)R.rot, half = rot / 2;
	const kv_vec<TY, VPL> own = *(const kv_vec<TY, VPL> *)(x + c0);
#pragma unroll
	for (int u = 0; u < VPL; u++) {
		const int c = c0 + u;
		y[u] = T::get(own.v[u]);
		if (c >= rot)
			continue;
		const bool first = R.layout == HIP_ROPE_PAIRS ? !(c & 1) : c < half;
		const int other = R.layout == HIP_ROPE_PAIRS ? c ^ 1 : first ? c + half : c - half;
		const double a = (double)y[u], b = (double)T::get(x[other]);
		y[u] = (float)(first ? a * cs[u] - b * sn[u] : a * cs[u] + b * sn[u]);
	}
}

/*
 * One workgroup: the call's rows in one tile of one sequence, for `per` kv
 * heads and as large a share of the q heads.  A wave takes a row at a time (a
 * head at a time where the tile has fewer than four rows), D / 64 channels a
 * lane; keys meet their group's scale in an xor-shuffle over its lanes, values
 * over the wave.  The value codes go to LDS, since one word holds eight rows'
 * codes of a channel: the words are put together from there, and a word that
 * has other rows' codes too is read first and keeps them.
 */
template <int D, int TY>
__global__ __launch_bounds__(KV_NT) void k_kv_append(
	kv_args a, hip_rope R, const typename kv_type<TY>::t *k, const typename kv_type<TY>::t *v,
	size_t kv_stride, const int32_t *pos, const typename kv_type<TY>::t *q, size_t q_stride,
	int heads, typename kv_type<TY>::t *q_out, size_t q_out_stride, int per, int tiles)
{
	typedef kv_type<TY> T;
	typedef kv_tile<D> L;
	constexpr int VPL = D / 64, LG = 32 / VPL, LW = 8 / VPL; /* lanes of a group, of a word */
	extern __shared__ uint8_t codes[]; /* [per][32][D] */
	const int groups = a.kv_heads / per + (a.kv_heads % per != 0);
	const int hg = blockIdx.x % groups, tb = blockIdx.x / groups % tiles;
	const int s = blockIdx.x / groups / tiles;
	const kv_seq sq = kv_sequence(a, s);
	const int p0 = max(0, sq.len - sq.n), t = p0 / KV_TILE + tb;
	const int lo = max(p0, t * KV_TILE), hi = min(sq.len, (t + 1) * KV_TILE);
	if (lo >= hi)
		return;
	const int h0 = hg * per, h1 = min(h0 + per, a.kv_heads);
	const int q0 = q ? heads * h0 / a.kv_heads : 0, q1 = q ? heads * h1 / a.kv_heads : 0;
	const int wave = threadIdx.x / WAVE, lane = threadIdx.x % WAVE, c0 = lane * VPL;
	const bool by_head = hi - lo < KV_NT / WAVE;

	for (int p = lo + (by_head ? 0 : wave); p < hi; p += by_head ? 1 : KV_NT / WAVE) {
		const int row = sq.row + p - (sq.len - sq.n), r = p % KV_TILE;
		double cs[VPL], sn[VPL];
#pragma unroll
		for (int u = 0; u < VPL; u++) {
			const int c = c0 + u, half = (int)R.rot / 2;
			const int i = R.layout == HIP_ROPE_PAIRS ? c / 2 : c % (half ? half : 1);
			if (u && R.layout == HIP_ROPE_PAIRS && (c & 1)) {
				cs[u] = cs[u - 1];
				sn[u] = sn[u - 1];
			} else if (c < (int)R.rot) {
				kv_turn(R, pos ? pos[row] : p, i, &cs[u], &sn[u]);
			}
		}
		const int step = by_head ? KV_NT / WAVE : 1;
		for (int h = h0 + (by_head ? wave : 0); h < h1; h += step) {
			uint8_t *tile = kv_tile_at<D>(a, s, h, t);
			if (!tile) {
				if (lane == 0)
					kv_error(a, HIP_KV_ERR_PAGE);
				continue;
			}
			float y[VPL], low, high;
			bool nan = false;
			kv_turned<TY, VPL>(k + row * kv_stride + h * D, c0, R, cs, sn, y);
			low = high = y[0];
#pragma unroll
			for (int u = 0; u < VPL; u++) {
				low = fminf(low, y[u]);
				high = fmaxf(high, y[u]);
				nan |= y[u] != y[u];
			}
			for (int o = LG / 2; o > 0; o >>= 1) {
				low = fminf(low, __shfl_xor(low, o, WAVE));
				high = fmaxf(high, __shfl_xor(high, o, WAVE));
			}
			const uint64_t group = ((1ull << LG) - 1) << (lane / LG * LG);
			if (__ballot(nan) & group)
				low = high = __builtin_nanf("");
			_Float16 d = low == low ? kv_scale(low, high) : (_Float16)low;
			float df = (float)d, inv = df == 0.0f ? 0.0f : 1.0f / fabsf(df);
			u32 w = 0;
#pragma unroll
			for (int u = 0; u < VPL; u++)
				w |= kv_rotr(kv_code(y[u], df, inv), 32 - kv_bit((c0 + u) % 8));
			for (int o = LW / 2; o > 0; o >>= 1)
				w |= (u32)__shfl_xor((int)w, o, WAVE);
			if (lane % LW == 0)
				((u32 *)tile)[L::k_word(r, c0)] = w;
			if (lane % LG == 0)
				((_Float16 *)(tile + L::K_SCALES))[r * L::G + c0 / 32] = d;

			/* the value row */
			const kv_vec<TY, VPL> x =
				*(const kv_vec<TY, VPL> *)(v + row * kv_stride + h * D + c0);
			nan = false;
			low = high = T::get(x.v[0]);
#pragma unroll
			for (int u = 0; u < VPL; u++) {
				y[u] = T::get(x.v[u]);
				low = fminf(low, y[u]);
				high = fmaxf(high, y[u]);
				nan |= y[u] != y[u];
			}
			for (int o = WAVE / 2; o > 0; o >>= 1) {
				low = fminf(low, __shfl_xor(low, o, WAVE));
				high = fmaxf(high, __shfl_xor(high, o, WAVE));
			}
			if (__ballot(nan))
				low = high = __builtin_nanf("");
			d = low == low ? kv_scale(low, high) : (_Float16)low;
			df = (float)d;
			inv = df == 0.0f ? 0.0f : 1.0f / fabsf(df);
#pragma unroll
			for (int u = 0; u < VPL; u++)
				codes[((h - h0) * KV_TILE + r) * D + c0 + u] =
					(uint8_t)kv_code(y[u], df, inv);
			if (lane == 0)
				((_Float16 *)(tile + L::V_SCALES))[r] = d;
		}
		for (int h = q0 + (by_head ? wave : 0); h < q1; h += step) {
			float y[VPL];
			kv_vec<TY, VPL> o;
			kv_turned<TY, VPL>(q + row * q_stride + h * D, c0, R, cs, sn, y);
#pragma unroll
			for (int u = 0; u < VPL; u++)
				o.v[u] = T::put(y[u]);
			__builtin_amdgcn_wave_barrier(); /* in place: the lanes' loads come first */
			*(kv_vec<TY, VPL> *)(q_out + row * q_out_stride + h * D + c0) = o;
		}
	}
	__syncthreads();

	const int r0 = lo % KV_TILE, r1 = r0 + hi - lo; /* the tile's rows of this call */
	for (int at = threadIdx.x; at < (h1 - h0) * 4 * D; at += KV_NT) {
		const int h = at / (4 * D), part = at / D % 4, c = at % D;
		u32 w = 0, mine = 0;
		for (int j = 0; j < 8; j++) {
			const int r = j / 4 * 16 + part * 4 + j % 4;
			if (r < r0 || r >= r1)
				continue;
			mine |= kv_rotr(15, 32 - kv_bit(j));
			w |= kv_rotr(codes[(h * KV_TILE + r) * D + c], 32 - kv_bit(j));
		}
		uint8_t *tile = mine ? kv_tile_at<D>(a, s, h0 + h, t) : NULL;
		if (!tile)
			continue;
		u32 *to = (u32 *)(tile + L::V_CODES) + L::v_word(part * 4, c);
		if (~mine)
			w |= *to & ~mine;
		*to = w;
	}
}

/* ---------------------------------------------------------------------- */
/* reading rows                                                           */
/* ---------------------------------------------------------------------- */

/* One workgroup: the batch's rows in one tile of one sequence, all heads;
 * a thread takes 8 channels of a row at a time. */
template <int D, int TY>
__global__ __launch_bounds__(KV_NT) void k_kv_read(kv_args a, typename kv_type<TY>::t *k,
						    typename kv_type<TY>::t *v, size_t stride,
						    int tiles)
{
	typedef kv_type<TY> T;
	typedef kv_tile<D> L;
	const int tb = blockIdx.x % tiles, s = blockIdx.x / tiles;
	const kv_seq sq = kv_sequence(a, s);
	const int p0 = max(0, sq.len - sq.n), t = p0 / KV_TILE + tb;
	const int lo = max(p0, t * KV_TILE), hi = min(sq.len, (t + 1) * KV_TILE);
	if (lo >= hi)
		return;
	for (int at = threadIdx.x; at < (hi - lo) * a.kv_heads * (D / 8); at += KV_NT) {
		const int c = at % (D / 8) * 8, h = at / (D / 8) % a.kv_heads;
		const int p = lo + at / (D / 8) / a.kv_heads, r = p % KV_TILE;
		const uint8_t *tile = kv_tile_at<D>(a, s, h, t);
		if (!tile) {
			kv_error(a, HIP_KV_ERR_PAGE);
			continue;
		}
		const size_t to = (sq.row + p - (sq.len - sq.n)) * stride + h * D + c;
		const u32 kw = ((const u32 *)tile)[L::k_word(r, c)];
		const float kd = (float)((const _Float16 *)(tile + L::K_SCALES))[r * L::G + c / 32];
		const float vd = (float)((const _Float16 *)(tile + L::V_SCALES))[r];
		const int bit = kv_bit(L::v_code(r));
		kv_vec<TY, 8> ko, vo;
#pragma unroll
		for (int j = 0; j < 8; j++) {
			const u32 vw = ((const u32 *)(tile + L::V_CODES))[L::v_word(r, c + j)];
			ko.v[j] = T::put((float)((int)(kv_rotr(kw, kv_bit(j)) & 15) - 8) * kd);
			vo.v[j] = T::put((float)((int)(kv_rotr(vw, bit) & 15) - 8) * vd);
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
	const size_t n = rows * (head_len - R->rot / 2);
	const int grid = (int)(n / KV_NT < 1 << 16 ? (n + KV_NT - 1) / KV_NT : 1 << 16);
	KV_DISPATCH_TYPE(type, TY, {
		typedef kv_type<TY>::t t;
		k_kv_rope<TY><<<grid, KV_NT, 0, (hipStream_t)stream>>>(
			(const t *)x, x_stride, (t *)out, out_stride, (int)rows, heads, head_len, *R, pos);
	})
	return (int)hipGetLastError();
}

extern "C" int kv_launch_append(const kv_args *a, int head_len, int type, const hip_rope *R,
				const void *k, const void *v, size_t kv_stride,
				const int32_t *pos, const void *q, size_t q_stride, int heads,
				void *q_out, size_t q_out_stride, void *stream)
{
	const hip_rope none = {0, HIP_ROPE_PAIRS, NULL, 1.0};
	const int tiles = kv_tiles_of(a->max_rows);
	/* one kv head a workgroup until the tiles alone fill the chip: the
	 * angles are then computed once for all heads */
	int per = 1;
	const int most = 32768 / (KV_TILE * head_len);
	while (per < most && per < a->kv_heads && (size_t)a->nseq * tiles * a->kv_heads / (2 * per) >= 1024)
		per *= 2;
	per = per < a->kv_heads ? per : a->kv_heads;
	const size_t grid = (size_t)a->nseq * tiles * ((a->kv_heads + per - 1) / per);
	const size_t lds = (size_t)per * KV_TILE * head_len;
	KV_DISPATCH_HEAD(head_len, D, KV_DISPATCH_TYPE(type, TY, {
		typedef kv_type<TY>::t t;
		k_kv_append<D, TY><<<dim3((unsigned)grid), KV_NT, lds, (hipStream_t)stream>>>(
			*a, R ? *R : none, (const t *)k, (const t *)v, kv_stride, pos, (const t *)q,
			q_stride, heads, (t *)q_out, q_out_stride, per, tiles);
	}))
	return (int)hipGetLastError();
}

extern "C" int kv_launch_read(const kv_args *a, int head_len, int type, void *k, void *v,
			      size_t stride, void *stream)
{
	const int tiles = kv_tiles_of(a->max_rows);
	const size_t grid = (size_t)a->nseq * tiles;
	KV_DISPATCH_HEAD(head_len, D, KV_DISPATCH_TYPE(type, TY, {
		typedef kv_type<TY>::t t;
		k_kv_read<D, TY><<<dim3((unsigned)grid), KV_NT, 0, (hipStream_t)stream>>>(
			*a, (t *)k, (t *)v, stride, tiles);
	}))
	return (int)hipGetLastError();
}
