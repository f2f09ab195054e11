/*
 * f8_mul.hip - products of e4m3 rows with e4m3 matrices that carry a scale for
 * 128 channels of a row and for 128 x 128 of a matrix (include/hip_f8.h), dense and
 * grouped by expert, plain and gated.
 *
 * A block of 128 channels is summed from 0 by the matrix cores, and joins the fp32
 * accumulator times the product of both scales.  The matrix rows are the
 * instruction's rows and the rows of X its columns, so that a lane has one row of X
 * and four neighbouring outputs, and needs one product of scales for 128 outputs.
 *
 * The 8-bit instruction takes the 128 channels at once, but adds up eight products
 * (a quarter of a lane's) after aligning them to the largest one's exponent and
 * cutting them off 13 bits below it: of normal values, sums are 1.3e-5 off, with some
 * channels 8 times larger than the rest 3e-5.  16-bit outputs are rounded by more than
 * that (1.7e-3 bf16, 2.1e-4 f16) and take it.  fp32 outputs take the 16-bit
 * instruction, whose sums of the same codes in f16 (exact) are 1.4e-8 off, at half
 * the rate and with a conversion for two codes.
 */
#include "kv_device.h"
#include "f8_internal.h"

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

/* 16 rows (columns) of an operand, 128 deep: lane l has row l % 16, and of the 128 any
 * 32 as long as both operands have the same */
template <bool EXACT> struct f8_operand;
template <> struct f8_operand<false> {
	i32x8 v;
	__device__ inline void set(i32x4 lo, i32x4 hi)
	{
		v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
	}
	/* the block's sum */
	__device__ static inline floatx4 mul(const f8_operand &a, const f8_operand &b)
	{
		return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.v, b.v, floatx4{0, 0, 0, 0}, 0, 0,
									0, 0, 0, 0);
	}
};
template <> struct f8_operand<true> {
	half8_t v[4];
	__device__ inline void set(i32x4 lo, i32x4 hi)
	{
#pragma unroll
		for (int i = 0; i < 4; i++)
#pragma unroll
			for (int j = 0; j < 2; j++) {
				const u32 w = i < 2 ? lo[2 * i + j] : hi[2 * i - 4 + j];
				const auto a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false);
				const auto b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true);
				v[i][4 * j] = a[0];
				v[i][4 * j + 1] = a[1];
				v[i][4 * j + 2] = b[0];
				v[i][4 * j + 3] = b[1];
			}
	}
	__device__ static inline floatx4 mul(const f8_operand &a, const f8_operand &b)
	{
		floatx4 y = {0, 0, 0, 0};
#pragma unroll
		for (int i = 0; i < 4; i++)
			y = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.v[i], b.v[i], y, 0, 0, 0);
		return y;
	}
};

/* The channels c .. c + 15 of a row's codes, zeros from k on */
__device__ static inline i32x4 f8_masked(i32x4 v, int c, int k)
{
#pragma unroll
	for (int i = 0; i < 4; i++) {
		const int left = k - c - 4 * i;
		v[i] = left >= 4 ? v[i] : left <= 0 ? 0 : v[i] & (int)(0xffffffffu >> (32 - 8 * left));
	}
	return v;
}

/* A tile's expert and rows of out */
struct f8_rows_of {
	int e, a, b; /* rows a .. b - 1, none if a >= b */
};

__device__ static inline int f8_clamp(int v, int lo, int hi)
{
	return v < lo ? lo : v > hi ? hi : v;
}

/* Tile `tile` of bt rows over all experts, whose tiles follow each other: 64 experts
 * at a time, a lane each, their tiles added up over the lanes. */
template <int BT>
__device__ static inline f8_rows_of f8_find(const f8_mul_args &A, int tile)
{
	if (!A.start)
		return f8_rows_of{0, tile * BT, tile * BT + BT < A.rows ? tile * BT + BT : A.rows};
	const int lane = threadIdx.x % 64;
	int before = 0;
	for (int e0 = 0; e0 < A.count; e0 += 64) {
		const int e = e0 + lane;
		int a = 0, b = 0;
		if (e < A.count) {
			a = f8_clamp(A.start[e], 0, A.rows);
			b = f8_clamp(A.start[e + 1], a, A.rows);
		}
		const int own = (b - a + BT - 1) / BT;
		int upto = own;
#pragma unroll
		for (int d = 1; d < 64; d *= 2) {
			const int o = __shfl_up(upto, d);
			upto += lane >= d ? o : 0;
		}
		const int first = before + upto - own;
		const unsigned long m = __ballot(tile >= first && tile < first + own);
		if (m) {
			const int l = __builtin_ctzl(m);
			const int at = __shfl(a, l) + (tile - __shfl(first, l)) * BT, end = __shfl(b, l);
			return f8_rows_of{e0 + l, at, at + BT < end ? at + BT : end};
		}
		before += __shfl(upto, 63);
	}
	return f8_rows_of{0, 0, 0};
}

__device__ static inline float f8_gate(float a, float b)
{
	return a / (1.0f + expf(-a)) * b;
}

/* N neighbouring outputs of a row, from n on */
template <int TY, int N>
__device__ static inline void f8_store(const f8_mul_args &A, int row, int n, float *y)
{
	typedef kv_type<TY> T;
	constexpr int PER = 16 / sizeof(typename T::t) < N ? 16 / sizeof(typename T::t) : N;
	typedef kv_vec<TY, PER> vec;
	typename T::t *o = (typename T::t *)A.out + row * A.out_stride + n;
	const typename T::t *p = (const typename T::t *)A.add + row * A.add_stride + n;
#pragma unroll
	for (int v0 = 0; v0 < N; v0 += PER) {
		if (n + v0 + PER <= A.n) {
			if (A.add) {
				const vec v = *(const vec *)(p + v0);
#pragma unroll
				for (int u = 0; u < PER; u++)
					y[v0 + u] += T::get(v.v[u]);
			}
			vec v;
#pragma unroll
			for (int u = 0; u < PER; u++)
				v.v[u] = T::put(y[v0 + u]);
			*(vec *)(o + v0) = v;
		} else {
#pragma unroll
			for (int u = 0; u < PER; u++)
				if (n + v0 + u < A.n)
					o[v0 + u] = T::put(A.add ? y[v0 + u] + T::get(p[v0 + u]) : y[v0 + u]);
		}
	}
}

/* 16 bytes a lane from its address to lds + 16 * lane, in flight until a wait that
 * the caller makes (moe_device.h's dma_dwordx4 with whole addresses) */
__device__ static inline void f8_dma16(const uint8_t *p, u32 lds)
{
	asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
		     :
		     : "v"(p), "{m0}"(__builtin_amdgcn_readfirstlane(lds))
		     : "memory");
}

/* the same, 4 bytes a lane */
__device__ static inline void f8_dma4(const float *p, u32 lds)
{
	asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, off"
		     :
		     : "v"(p), "{m0}"(__builtin_amdgcn_readfirstlane(lds))
		     : "memory");
}

/* All waves have come here, their LDS reads are done, and of each one's loads
 * all but the last N have arrived */
template <int N>
__device__ static inline void f8_meet()
{
	static_assert(N >= 0 && N < 64, "vmcnt is six bits");
	asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

#ifndef F8_SCHEDULE
#define F8_SCHEDULE
#endif
/*
 * Tiles of 16 NB WT rows of X and 16 NA WN rows of W (gated: half of them W's, half
 * up's), a wave 16 NB by 16 NA of them.  A step is a block of 128 channels, all rows'
 * 128 bytes and X's scales in one of STAGES buffers, filled by loads that go past the
 * registers, STAGES - 1 steps ahead.
 *
 * A row's 128 bytes are eight pieces of 16; piece p lies at place p ^ (row % 8), so
 * that the 16 rows whose same piece an operand's read takes meet no bank twice.  Row
 * i of an operand's 16 is the output that gives a lane its 4 NA neighbouring ones.
 */
template <int TY, bool GATED, int NA, int NB, int WN, int WT, int STAGES>
__global__ __launch_bounds__(64 * WN * WT) void k_f8_tile(f8_mul_args A, int n_tiles, int row_tiles)
{
	constexpr int M = GATED ? 2 : 1, FA = NA / M; /* operands of one matrix */
	constexpr int BN = 16 * NA * WN, BT = 16 * NB * WT, NO = BN / M;
	constexpr int NW = WN * WT, SLOTS = (BN + BT) / 8 / NW, SCALES = BT < 64 ? 64 : BT;
	constexpr int BYTES = (BN + BT) * HIP_F8_BLOCK + SCALES * 4 + 256;
	static_assert((BN + BT) / 8 % NW == 0 && HIP_F8_BLOCK % (16 * FA) == 0, "whole loads, one scale");
	static_assert(SCALES / 64 < NW && WN * M <= 64, "a wave is left for W's scales");
	typedef f8_operand<TY == HIP_F8_F32> operand;
	__shared__ __attribute__((aligned(16))) uint8_t lds[STAGES * BYTES];

	const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
	const int wn = wave % WN, wt = wave / WN;
	/* Workgroups go to the eight XCDs in turn: each takes a stretch of the tiles, in
	 * groups of 8 row tiles that share what the L2 holds of W. */
	const int grid = n_tiles * row_tiles, xcd = blockIdx.x % 8;
	const int id = xcd * (grid / 8) + (xcd < grid % 8 ? xcd : grid % 8) + blockIdx.x / 8;
	const int group = id / (8 * n_tiles), g0 = group * 8;
	const int many = row_tiles - g0 < 8 ? row_tiles - g0 : 8;
	const int in = id - group * 8 * n_tiles;
	const int tile = g0 + in % many, n0 = in / many * NO;

	f8_rows_of R = f8_find<BT>(A, tile);
	R.e = __builtin_amdgcn_readfirstlane(R.e);
	R.a = __builtin_amdgcn_readfirstlane(R.a);
	R.b = __builtin_amdgcn_readfirstlane(R.b);
	if (R.a >= R.b)
		return;

	/* what this wave loads: slots of eight rows */
	const int piece = ((lane % 8) ^ (lane / 8)) * 16, last = (A.k - 1) & ~15;
	const uint8_t *p[SLOTS];
#pragma unroll
	for (int i = 0; i < SLOTS; i++) {
		const int s = wave + i * NW, row = s * 8 + lane / 8;
		if (row < BN) {
			const int j = row % (16 * NA), m = j / (16 * FA), f = j / 16 % FA, r = j % 16;
			int n = n0 + row / (16 * NA) * (16 * FA) + r / 4 * (4 * FA) + f * 4 + r % 4;
			n = n < A.n ? n : A.n - 1;
			p[i] = (m ? A.w[M - 1] + R.e * A.w_step[M - 1] + n * A.w_stride[M - 1]
				  : A.w[0] + R.e * A.w_step[0] + n * A.w_stride[0]);
		} else {
			int x = R.a + row - BN;
			x = x < R.b ? x : R.b - 1;
			x = A.from ? A.from[x] : x;
			x = (unsigned)x < (unsigned)A.x_rows ? x : 0;
			p[i] = A.x + x * A.x_stride;
		}
	}
	/* and of the scales: X's 64 at a time, then W's, one for each wn and matrix */
	const float *ps;
	long ps_step;
	const int sslot = wave < SCALES / 64 ? wave : SCALES / 64;
	if (sslot < SCALES / 64) {
		int x = R.a + sslot * 64 + lane;
		x = x < R.b ? x : R.b - 1;
		x = A.from ? A.from[x] : x;
		ps = A.xs + ((unsigned)x < (unsigned)A.x_rows ? x : 0);
		ps_step = A.xs_stride;
	} else {
		const int m = lane % M;
		int n = n0 + lane / M % WN * 16 * FA;
		n = n < A.n ? n : A.n - 1;
		ps = A.ws[m] + R.e * A.ws_step[m] + n / HIP_F8_BLOCK * A.ws_stride[m];
		ps_step = 1;
	}
	const int blocks = (A.k + HIP_F8_BLOCK - 1) / HIP_F8_BLOCK;
	const u32 base = lds_addr(lds);
	auto load = [&](int kb, int stage) {
		int c = kb * HIP_F8_BLOCK + piece;
		c = c < last ? c : last; /* nothing past the row's last 16 that hold any is read */
		const u32 to = base + stage * BYTES;
#pragma unroll
		for (int i = 0; i < SLOTS; i++)
			f8_dma16(p[i] + c, to + (wave + i * NW) * 1024);
		f8_dma4(ps + kb * ps_step, to + (BN + BT) * HIP_F8_BLOCK + sslot * 256);
	};
	floatx4 acc[NA][NB] = {};
#pragma unroll
	for (int s = 0; s < STAGES - 1; s++)
		load(s < blocks ? s : blocks - 1, s);
	int stage = 0;
	const int place = ((lane / 16) ^ (lane % 8)) * 16;
	for (int kb = 0; kb < blocks; kb++) {
		f8_meet<(STAGES - 2) * (SLOTS + 1)>();
		const int ahead = kb + STAGES - 1;
		load(ahead < blocks ? ahead : blocks - 1, stage == 0 ? STAGES - 1 : stage - 1);
		uint8_t *buf = lds + stage * BYTES;
		if ((kb + 1) * HIP_F8_BLOCK > A.k) { /* the last block's rest: zeros */
			for (int i = threadIdx.x; i < (BN + BT) * 8; i += 64 * NW) {
				const int c = kb * HIP_F8_BLOCK + ((i % 8) ^ (i / 8 % 8)) * 16;
				i32x4 *q = (i32x4 *)(buf + i * 16);
				if (c + 16 > A.k)
					*q = f8_masked(*q, c, A.k);
			}
			f8_meet<63>();
		}
		const float *sx = (const float *)(buf + (BN + BT) * HIP_F8_BLOCK);
		float s[M][NB];
#pragma unroll
		for (int b = 0; b < NB; b++)
#pragma unroll
			for (int m = 0; m < M; m++)
				s[m][b] = sx[(wt * NB + b) * 16 + lane % 16] * sx[SCALES + wn * M + m];
		operand x[NB], w[2];
		const uint8_t *xb = buf + (BN + wt * 16 * NB + lane % 16) * HIP_F8_BLOCK;
		const uint8_t *wb = buf + (wn * 16 * NA + lane % 16) * HIP_F8_BLOCK;
		w[0].set(*(const i32x4 *)(wb + place), *(const i32x4 *)(wb + (place ^ 64)));
#pragma unroll
		for (int b = 0; b < NB; b++)
			x[b].set(*(const i32x4 *)(xb + b * 2048 + place), *(const i32x4 *)(xb + b * 2048 + (place ^ 64)));
		/* the sums of operand a are made while those of a - 1 join the accumulators */
		floatx4 y[2][NB];
#pragma unroll
		for (int a = 0; a <= NA; a++) {
			if (a + 1 < NA)
				w[(a + 1) % 2].set(*(const i32x4 *)(wb + (a + 1) * 2048 + place),
						   *(const i32x4 *)(wb + (a + 1) * 2048 + (place ^ 64)));
#pragma unroll
			for (int b = 0; b < NB; b++) {
				if (a < NA)
					y[a % 2][b] = operand::mul(w[a % 2], x[b]);
				if (a > 0)
#pragma unroll
					for (int u = 0; u < 4; u++)
						acc[a - 1][b][u] = __builtin_fmaf(y[(a - 1) % 2][b][u], s[(a - 1) / FA][b],
										  acc[a - 1][b][u]);
			}
		}
		F8_SCHEDULE
		stage = stage + 1 == STAGES ? 0 : stage + 1;
	}
	f8_meet<0>(); /* no load outlives the workgroup's LDS */
	const int n = n0 + wn * 16 * FA + lane / 16 * (4 * FA);
#pragma unroll
	for (int b = 0; b < NB; b++) {
		const int r = R.a + (wt * NB + b) * 16 + lane % 16;
		if (r >= R.b || n >= A.n)
			continue;
		const bool bad = A.from && (unsigned)A.from[r] >= (unsigned)A.x_rows;
		float y[4 * FA];
#pragma unroll
		for (int f = 0; f < FA; f++)
#pragma unroll
			for (int u = 0; u < 4; u++) {
				y[4 * f + u] = GATED ? f8_gate(acc[f][b][u], acc[NA - FA + f][b][u]) : acc[f][b][u];
				if (bad)
					y[4 * f + u] = __builtin_nanf("");
			}
		f8_store<TY, 4 * FA>(A, r, n, y);
	}
}

/* the tiles of a type and form: NA, NB, WN, WT, STAGES */
#define F8_BIG 8, 4, 2, 4, 2     /* 256 x 256 */
#define F8_BIG_F32 4, 4, 2, 4, 2 /* 128 x 256 */
#define F8_SMALL 2, 4, 4, 1, 3   /* 128 x 64 */
#define F8_SMALL_F32 2, 2, 4, 2, 3 /* 128 x 64 */

void f8_mul_plan(const f8_mul_args *a, f8_plan *p)
{
	const size_t rows = (size_t)a->rows, n = (size_t)a->n;
	const size_t per = a->start ? (rows + (size_t)a->count - 1) / (size_t)a->count : rows;
	p->big = per > 128;
	p->bt = p->big ? 256 : 64;
	p->bn = p->big && p->type != HIP_F8_F32 ? 256 : 128;
	if (a->w[1])
		p->bn /= 2;
	p->threads = p->big || p->type == HIP_F8_F32 ? 512 : 256;
	p->n_tiles = (n + (size_t)p->bn - 1) / (size_t)p->bn;
	p->row_tiles = (rows + (size_t)p->bt - 1) / (size_t)p->bt;
	if (a->start) /* every expert may end with a tile that is not full */
		p->row_tiles = rows / (size_t)p->bt + (rows < (size_t)a->count ? rows : (size_t)a->count);
}

template <int TY, int... FORM>
static void tile_typed(const f8_mul_args *a, const f8_plan *p, hipStream_t s)
{
	const size_t grid = p->row_tiles * p->n_tiles;
	if (a->w[1])
		k_f8_tile<TY, true, FORM...><<<grid, p->threads, 0, s>>>(*a, (int)p->n_tiles, (int)p->row_tiles);
	else
		k_f8_tile<TY, false, FORM...><<<grid, p->threads, 0, s>>>(*a, (int)p->n_tiles, (int)p->row_tiles);
}

int f8_launch_mul(const f8_mul_args *a, const f8_plan *p, void *stream)
{
	hipStream_t s = (hipStream_t)stream;
	if (p->type == HIP_F8_F32)
		p->big ? tile_typed<HIP_F8_F32, F8_BIG_F32>(a, p, s) : tile_typed<HIP_F8_F32, F8_SMALL_F32>(a, p, s);
	else if (p->type == HIP_F8_F16)
		p->big ? tile_typed<HIP_F8_F16, F8_BIG>(a, p, s) : tile_typed<HIP_F8_F16, F8_SMALL>(a, p, s);
	else
		p->big ? tile_typed<HIP_F8_BF16, F8_BIG>(a, p, s) : tile_typed<HIP_F8_BF16, F8_SMALL>(a, p, s);
	return hipGetLastError();
}
