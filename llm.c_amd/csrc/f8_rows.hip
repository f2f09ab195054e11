/*
 * f8_rows.hip - rows into 8-bit floating point, pairs of tokens and experts by
 * expert, and the experts' outputs back to tokens (include/hip_f8.h has the
 * formulas).
 */
#include "kv_device.h"
#include "f8_internal.h"

#define QUANT_CHANNELS 512 /* of a row, by one wave */

/*
 * The e4m3 code of x / s, ties to even, as a float that the conversion rounds to
 * it.  q is within a step of x / s in fp32, r = 1 / s; its remainder x - q s is exact.
 * Rounding q instead of x / s differs only where q is halfway between two codes (19
 * low bits of zero) and the remainder is not 0: then q moves a step to the
 * remainder's side.  Scales of 2^-96 and more keep the remainder out of the
 * subnormal numbers' steps.
 */
__device__ static inline float f8_quotient(float x, float s, float r)
{
	const float q0 = x * r;
	const float q = __builtin_fmaf(__builtin_fmaf(-q0, s, x), r, q0);
	const float rest = __builtin_fmaf(-q, s, x);
	u32 b = __builtin_bit_cast(u32, q);
	if (!(b & 0x7ffff) && rest != 0.0f)
		b += (int)(b ^ __builtin_bit_cast(u32, rest)) < 0 ? -1 : 1;
	return __builtin_bit_cast(float, b);
}

/*
 * R rows a wave, 512 channels of each; 16 bytes a lane and load, so that the 128
 * channels of a scale are 32 (fp32) or 16 lanes.  Two rows a wave, whose loads are in
 * flight together, where that leaves 2048 workgroups (28 -> 24 us for 8192 x 4096 bf16, 4.2 TB/s;
 * fp32 33 us, 5.1 TB/s); 16 rows of 4096 take 3.2 us, the launch and one load's latency.
 * Stores that pass the caches took 22 us, and the product after them 3 us longer (8192 rows by
 * 4096 x 1024).
 */
template <int TY, int R>
__global__ __launch_bounds__(F8_ROW_THREADS) void k_f8_quantize(
	const typename kv_type<TY>::t *__restrict__ x, size_t x_stride, hip_f8_rows X)
{
	typedef kv_type<TY> T;
	constexpr int N = 16 / sizeof(typename T::t), LANES = HIP_F8_BLOCK / N;
	constexpr int STEPS = QUANT_CHANNELS / (64 * N);
	typedef kv_vec<TY, N> vec;
	const size_t parts = (X.k + QUANT_CHANNELS - 1) / QUANT_CHANNELS;
	const size_t part = blockIdx.x % parts;
	const size_t r0 = (blockIdx.x / parts * (F8_ROW_THREADS / 64) + threadIdx.x / 64) * R;
	const int lane = threadIdx.x % 64;
	vec v[R][STEPS];
#pragma unroll
	for (int i = 0; i < R; i++)
#pragma unroll
		for (int j = 0; j < STEPS; j++) {
			const size_t c = part * QUANT_CHANNELS + (j * 64 + lane) * N;
			if (r0 + i < X.rows && c < X.k)
				v[i][j] = *(const vec *)(x + (r0 + i) * x_stride + c);
		}
#pragma unroll
	for (int i = 0; i < R; i++)
#pragma unroll
		for (int j = 0; j < STEPS; j++) {
			const size_t c = part * QUANT_CHANNELS + (j * 64 + lane) * N;
			float y[N];
			u32 top = 0;
#pragma unroll
			for (int u = 0; u < N; u++) {
				y[u] = c + u < X.k ? T::get(v[i][j].v[u]) : 0.0f;
				const u32 b = __builtin_bit_cast(u32, y[u]) & 0x7fffffff;
				top = top > b ? top : b; /* NaN above infinity above numbers */
			}
#pragma unroll
			for (int d = 1; d < LANES; d *= 2) {
				const u32 b = __shfl_xor(top, d);
				top = top > b ? top : b;
			}
			if (r0 + i >= X.rows || c >= ((X.k + 15) & ~(size_t)15))
				continue;
			const bool bad = top >= 0x7f800000;
			const float m = __builtin_bit_cast(float, top) / 448.0f;
			const float s = m > 0x1p-96f ? m : 0x1p-96f;
			const float rec = 1.0f / s;
			u32 w[N / 4];
#pragma unroll
			for (int u = 0; u < N; u += 4) {
				int p = 0;
				p = __builtin_amdgcn_cvt_pk_fp8_f32(f8_quotient(y[u], s, rec),
								    f8_quotient(y[u + 1], s, rec), p, false);
				p = __builtin_amdgcn_cvt_pk_fp8_f32(f8_quotient(y[u + 2], s, rec),
								    f8_quotient(y[u + 3], s, rec), p, true);
				w[u / 4] = bad ? 0 : p;
			}
			u32 *o = (u32 *)(X.codes + (r0 + i) * X.stride + c);
			if constexpr (N == 4)
				*o = w[0];
			else
				*(u32x2 *)o = u32x2{w[0], w[1]};
			if (lane % LANES == 0)
				X.scale[c / HIP_F8_BLOCK * X.scale_stride + r0 + i] =
					bad ? __builtin_nanf("") : s;
		}
}

#define QUANT_ROWS 2

size_t f8_quantize_grid(size_t rows, size_t k)
{
	return (rows + 3) / 4 * ((k + QUANT_CHANNELS - 1) / QUANT_CHANNELS);
}

template <int TY>
static void quantize_typed(const void *x, size_t x_stride, const hip_f8_rows *X, hipStream_t s)
{
	typedef typename kv_type<TY>::t t;
	const size_t one = f8_quantize_grid(X->rows, X->k);
	if (one < 4096) {
		k_f8_quantize<TY, 1><<<one, F8_ROW_THREADS, 0, s>>>((const t *)x, x_stride, *X);
	} else {
		const size_t parts = (X->k + QUANT_CHANNELS - 1) / QUANT_CHANNELS;
		k_f8_quantize<TY, QUANT_ROWS><<<(X->rows + 4 * QUANT_ROWS - 1) / (4 * QUANT_ROWS) * parts,
						F8_ROW_THREADS, 0, s>>>((const t *)x, x_stride, *X);
	}
}

int f8_launch_quantize(int type, const void *x, size_t x_stride, const hip_f8_rows *X, void *stream)
{
	hipStream_t s = (hipStream_t)stream;
	if (type == HIP_F8_F32)
		quantize_typed<HIP_F8_F32>(x, x_stride, X, s);
	else if (type == HIP_F8_F16)
		quantize_typed<HIP_F8_F16>(x, x_stride, X, s);
	else
		quantize_typed<HIP_F8_BF16>(x, x_stride, X, s);
	return hipGetLastError();
}

/*
 * A workgroup an expert, and one more for the pairs without: each reads all ids, a
 * wave a stretch of up to 4096 of each 65536.  The counts of smaller ids and of its own
 * give the expert's first row and each wave's, ballots the rows inside a wave, so that
 * the order is the pairs' and nothing is shared between workgroups.  Up to 65536 pairs
 * are read once and stay in registers.  It is bound by its own chain: 8192 tokens of 8
 * slots take 17 us, ten for the launch and 256 KB of ids in every workgroup, three each for
 * counting, ranking and the scattered stores.  (Waves' loads next to each other, or
 * starting at another place in each workgroup, took as long.)
 */
#define SORT_WAVES 16
#define SORT_LOADS 16 /* of 4 ids a lane */

/* `loads` times 256 ids from a on; what is past the pairs is no expert's.  There is a
 * pair at least. */
__device__ static inline void sort_get(dw4 (&v)[SORT_LOADS], const u32 *__restrict__ ids, u32 a,
				       int loads, u32 pairs)
{
	const u32 i0 = a + threadIdx.x % 64 * 4;
	if (a + loads * 256 <= pairs) {
#pragma unroll
		for (int j = 0; j < SORT_LOADS; j++)
			if (j < loads)
				v[j] = *(const dw4 *)(ids + (i0 + j * 256));
		return;
	}
#pragma unroll
	for (int j = 0; j < SORT_LOADS; j++)
		if (j < loads)
#pragma unroll
			for (u32 u = 0; u < 4; u++) {
				const u32 i = i0 + j * 256 + u;
				const u32 id = ids[i < pairs ? i : pairs - 1];
				v[j].v[u] = i < pairs ? id : 0xffffffffu;
			}
}

/* A pair's token is pair * magic >> (32 + shift), magic = 2^(32 + shift) / topk rounded up
 * and 2^shift < topk <= 2^(shift + 1): magic is less than a whole too large, which moves
 * the quotient by less than 2^31 / 2^(32 + shift) < 1 / topk (topk 1: magic 0). */
__global__ __launch_bounds__(SORT_WAVES * 64) void k_f8_sort(
	const u32 *__restrict__ ids, u32 pairs, int loads, u32 magic, int shift, int experts,
	int *__restrict__ start, int *__restrict__ from, int *__restrict__ pos)
{
	__shared__ int n_own[SORT_WAVES], n_less[SORT_WAVES];
	const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), waves = blockDim.x / 64;
	const int lane = threadIdx.x % 64;
	const u32 stretch = loads * 256, chunk = waves * stretch, chunks = (pairs + chunk - 1) / chunk;
	const u32 e = blockIdx.x;
	if ((int)e == experts) {
		for (u32 i = threadIdx.x; i < pairs; i += blockDim.x)
			if (ids[i] >= e)
				pos[i] = -1;
		return;
	}
	dw4 v[SORT_LOADS];
	int less = 0;
	/* the chunks from the last to the first, which stays in the registers */
	for (u32 c = chunks; c-- > 0;) {
		const u32 a = c * chunk + wave * stretch;
		sort_get(v, ids, a, loads, pairs);
#pragma unroll
		for (int j = 0; j < SORT_LOADS; j++)
			if (j < loads) {
#pragma unroll
				for (int u = 0; u < 4; u++)
					less += __popcll(__ballot(v[j].v[u] < e));
			}
	}
	const unsigned long lower = (1ul << lane) - 1;
	int first = 0, rows = 0; /* the expert's first, and its rows of the chunks before */
	for (u32 c = 0; c < chunks; c++) {
		const u32 a = c * chunk + wave * stretch;
		if (c > 0)
			sort_get(v, ids, a, loads, pairs);
		int own = 0;
#pragma unroll
		for (int j = 0; j < SORT_LOADS; j++)
			if (j < loads) {
#pragma unroll
				for (int u = 0; u < 4; u++)
					own += __popcll(__ballot(v[j].v[u] == e));
			}
		if (lane == 0) {
			n_own[wave] = own;
			n_less[wave] = less;
		}
		__syncthreads();
		int before = 0, all = 0;
		for (int w = 0; w < waves; w++) {
			first += c == 0 ? n_less[w] : 0;
			before += w < wave ? n_own[w] : 0;
			all += n_own[w];
		}
		int row = first + rows + before;
		rows += all;
#pragma unroll
		for (int j = 0; j < SORT_LOADS; j++)
			if (j < loads) {
				int at = row;
				bool mine[4];
#pragma unroll
				for (int u = 0; u < 4; u++) {
					/* compared again: the masks of all loads have no room */
					asm volatile("" : "+v"(v[j].v[u]));
					mine[u] = v[j].v[u] == e;
					const unsigned long m = __ballot(mine[u]);
					at += __popcll(m & lower);
					row += __popcll(m);
				}
#pragma unroll
				for (int u = 0; u < 4; u++)
					if (mine[u]) {
						const u32 i = a + j * 256 + lane * 4 + u;
						from[at] = magic ? (int)(__umulhi(i, magic) >> shift) : (int)i;
						pos[i] = at++;
					}
			}
		__syncthreads(); /* before the next chunk's counts */
	}
	if (threadIdx.x == 0) {
		start[e] = first;
		if ((int)e == experts - 1)
			start[experts] = first + rows;
	}
}

int f8_launch_sort(const uint32_t *ids, int tokens, int topk, int experts, int32_t *start,
		   int32_t *from, int32_t *pos, void *stream)
{
	const long pairs = (long)tokens * topk;
	/* as few loads a wave as sixteen waves allow */
	long loads = (pairs + SORT_WAVES * 256 - 1) / (SORT_WAVES * 256);
	loads = loads < 1 ? 1 : loads > SORT_LOADS ? SORT_LOADS : loads;
	long waves = (pairs + loads * 256 - 1) / (loads * 256);
	waves = waves < 1 ? 1 : waves > SORT_WAVES ? SORT_WAVES : waves;
	int shift = 0;
	while ((2 << shift) < topk)
		shift++;
	const u32 magic = topk == 1 ? 0 : (u32)((((uint64_t)1 << (32 + shift)) + topk - 1) / topk);
	k_f8_sort<<<experts + 1, 64 * waves, 0, (hipStream_t)stream>>>(ids, (u32)pairs, (int)loads, magic, shift,
									experts, start, from, pos);
	return hipGetLastError();
}

/* 16 bytes of a token's values a thread; `lanes` threads (a power of two) a token.  Four
 * rows' loads in flight a thread: 8192 tokens of 8 slots, a quarter without a row, 2048 bf16 values:
 * 57 us, 4.7 TB/s. */
template <int TY>
__global__ __launch_bounds__(F8_ROW_THREADS) void k_f8_combine(
	const typename kv_type<TY>::t *__restrict__ y, size_t y_stride, int y_rows,
	const int *__restrict__ pos, const float *__restrict__ w, int tokens, int topk, int n,
	const typename kv_type<TY>::t *add, size_t add_stride, typename kv_type<TY>::t *out,
	size_t out_stride, int lanes, int parts)
{
	typedef kv_type<TY> T;
	constexpr int N = 16 / sizeof(typename T::t), AT_ONCE = 4;
	typedef kv_vec<TY, N> vec;
	const size_t t = (size_t)(blockIdx.x / parts) * (F8_ROW_THREADS / lanes) + threadIdx.x / lanes;
	const size_t c = ((size_t)(blockIdx.x % parts) * lanes + threadIdx.x % lanes) * N;
	if (t >= (size_t)tokens || c >= (size_t)n)
		return;
	float sum[N];
	if (add) {
		const vec v = *(const vec *)(add + t * add_stride + c);
#pragma unroll
		for (int u = 0; u < N; u++)
			sum[u] = T::get(v.v[u]);
	} else {
#pragma unroll
		for (int u = 0; u < N; u++)
			sum[u] = 0.0f;
	}
	for (int s0 = 0; s0 < topk; s0 += AT_ONCE) {
		vec v[AT_ONCE];
		float f[AT_ONCE];
		bool here[AT_ONCE];
#pragma unroll
		for (int s = 0; s < AT_ONCE; s++) {
			const int p = s0 + s < topk ? pos[t * topk + s0 + s] : -1;
			here[s] = p >= 0 && p < y_rows;
			if (here[s]) {
				f[s] = w[t * topk + s0 + s];
				v[s] = *(const vec *)(y + (size_t)p * y_stride + c);
			}
		}
#pragma unroll
		for (int s = 0; s < AT_ONCE; s++)
			if (here[s])
#pragma unroll
				for (int u = 0; u < N; u++)
					sum[u] = __builtin_fmaf(f[s], T::get(v[s].v[u]), sum[u]);
	}
	typename T::t *o = out + t * out_stride + c;
	if (c + N <= (size_t)n) {
		vec v;
#pragma unroll
		for (int u = 0; u < N; u++)
			v.v[u] = T::put(sum[u]);
		*(vec *)o = v;
	} else {
#pragma unroll
		for (int u = 0; u < N; u++)
			if (c + u < (size_t)n)
				o[u] = T::put(sum[u]);
	}
}

static int combine_lanes(int type, size_t n)
{
	const size_t vecs = type == HIP_F8_F32 ? (n + 3) / 4 : (n + 7) / 8;
	int lanes = 1;
	while (lanes < F8_ROW_THREADS && (size_t)lanes < vecs)
		lanes *= 2;
	return lanes;
}

size_t f8_combine_grid(int type, size_t tokens, size_t n)
{
	const size_t lanes = (size_t)combine_lanes(type, n), per = F8_ROW_THREADS / lanes;
	const size_t vecs = type == HIP_F8_F32 ? (n + 3) / 4 : (n + 7) / 8;
	return (tokens + per - 1) / per * ((vecs + lanes - 1) / lanes);
}

template <int TY>
static void combine_typed(const void *y, size_t y_stride, int y_rows, const int *pos, const float *w,
			  int tokens, int topk, int n, const void *add, size_t add_stride, void *out,
			  size_t out_stride, hipStream_t s)
{
	typedef typename kv_type<TY>::t t;
	constexpr int N = 16 / sizeof(t);
	const int lanes = combine_lanes(TY, (size_t)n);
	const int parts = (n + N * lanes - 1) / (N * lanes);
	k_f8_combine<TY><<<f8_combine_grid(TY, (size_t)tokens, (size_t)n), F8_ROW_THREADS, 0, s>>>(
		(const t *)y, y_stride, y_rows, pos, w, tokens, topk, n, (const t *)add, add_stride,
		(t *)out, out_stride, lanes, parts);
}

int f8_launch_combine(int type, const void *y, size_t y_stride, int y_rows, const int32_t *pos,
		      const float *w, int tokens, int topk, int n, const void *add, size_t add_stride,
		      void *out, size_t out_stride, void *stream)
{
	hipStream_t s = (hipStream_t)stream;
	if (type == HIP_F8_F32)
		combine_typed<HIP_F8_F32>(y, y_stride, y_rows, pos, w, tokens, topk, n, add, add_stride, out,
					  out_stride, s);
	else if (type == HIP_F8_F16)
		combine_typed<HIP_F8_F16>(y, y_stride, y_rows, pos, w, tokens, topk, n, add, add_stride, out,
					  out_stride, s);
	else
		combine_typed<HIP_F8_BF16>(y, y_stride, y_rows, pos, w, tokens, topk, n, add, add_stride, out,
					   out_stride, s);
	return hipGetLastError();
}
