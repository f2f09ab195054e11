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

/* An operand's codes as they lie in LDS, at p and at the place of the piece that is
 * four further */
struct f8_raw {
	i32x8 v;
	__device__ inline void get(const uint8_t *p, int place)
	{
		const i32x4 lo = *(const i32x4 *)p, hi = *(const i32x4 *)(p + (place & 64 ? -64 : 64));
		v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
	}
	/* the same from two places */
	__device__ inline void get2(const uint8_t *p, const uint8_t *q)
	{
		const i32x4 lo = *(const i32x4 *)p, hi = *(const i32x4 *)q;
		v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
	}
	/* zeros from channel k on, of c .. c + 15 and c + 64 .. c + 79 */
	__device__ inline void cut(int c, int k)
	{
		const i32x4 lo = f8_masked(__builtin_shufflevector(v, v, 0, 1, 2, 3), c, k);
		const i32x4 hi = f8_masked(__builtin_shufflevector(v, v, 4, 5, 6, 7), c + 64, k);
		v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
	}
};

/* 16 rows (columns) of an operand, 128 deep: lane l has row l % 16, and of the 128 any
 * 32 as long as both operands have the same */
template <bool EXACT> struct f8_operand;
template <> struct f8_operand<false> {
	i32x8 v;
	__device__ inline void set(const f8_raw &r)
	{
		v = r.v;
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
	__device__ inline void set(const f8_raw &r)
	{
#pragma unroll
		for (int i = 0; i < 4; i++)
#pragma unroll
			for (int j = 0; j < 2; j++) {
				const u32 w = r.v[2 * i + j];
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

/* A tile's expert and rows of out */
struct f8_rows_of {
	int e, a, b; /* rows a .. b - 1, none if a >= b */
};

__device__ static inline int f8_clamp(int v, int lo, int hi)
{
	return v < lo ? lo : v > hi ? hi : v;
}

/* The lane, anew: what is worked out from it between two tiles does not take registers
 * from the steps (the compiler's own hoisting spilled seven, 938 -> 1107 us for 16384 channels) */
__device__ static inline int f8_lane()
{
	int l = threadIdx.x % 64;
	asm volatile("" : "+v"(l));
	return l;
}

/* 64 experts from e0 on, a lane each: its rows a .. b - 1, its tiles of BT rows, and those
 * of the lanes up to it */
template <int BT> struct f8_scan {
	int a, b, own, upto;
	__device__ inline void get(const f8_mul_args &A, const int *start, int e0)
	{
		const int lane = f8_lane(), e = e0 + lane;
		a = b = 0;
		if (e < A.count) {
			a = f8_clamp(start[e], 0, A.rows);
			b = f8_clamp(start[e + 1], a, A.rows);
		}
		own = upto = (b - a + BT - 1) / BT;
#pragma unroll
		for (int d = 1; d < 64; d *= 2) {
			const int o = __shfl_up(upto, d);
			upto += lane >= d ? o : 0;
		}
	}
	__device__ inline int all() const { return __builtin_amdgcn_readlane(upto, 63); }
	/* tile `tile` of these, the first of which is tile `before` */
	__device__ inline bool find(int tile, int before, int e0, f8_rows_of &R) const
	{
		const int first = before + upto - own;
		const unsigned long m = __ballot(tile >= first && tile < first + own);
		if (!m)
			return false;
		const int l = __builtin_ctzl(m), end = __builtin_amdgcn_readlane(b, l);
		const int at = __builtin_amdgcn_readlane(a, l) + (tile - __builtin_amdgcn_readlane(first, l)) * BT;
		R = f8_rows_of{e0 + l, at, at + BT < end ? at + BT : end};
		return true;
	}
};

/* Tiles of BT rows over all experts, whose tiles follow each other; without experts the
 * host's count */
template <int BT>
__device__ static inline int f8_row_tiles(const f8_mul_args &A, const int *start, int row_tiles)
{
	if (!A.start)
		return row_tiles;
	f8_scan<BT> s;
	int n = 0;
	for (int e0 = 0; e0 < A.count; e0 += 64) {
		s.get(A, start, e0);
		n += s.all();
	}
	return n;
}

/* Rows of such a tile, none past the last */
template <int BT>
__device__ static inline f8_rows_of f8_find(const f8_mul_args &A, const int *start, int tile)
{
	f8_rows_of R = {0, 0, 0};
	if (!A.start) {
		R.a = tile * BT;
		R.b = R.a + BT < A.rows ? R.a + BT : A.rows;
		return R;
	}
	f8_scan<BT> s;
	int before = 0;
	for (int e0 = 0; e0 < A.count; e0 += 64) {
		s.get(A, start, e0);
		if (s.find(tile, before, e0, R))
			break;
		before += s.all();
	}
	return f8_rows_of{__builtin_amdgcn_readfirstlane(R.e), __builtin_amdgcn_readfirstlane(R.a),
			  __builtin_amdgcn_readfirstlane(R.b)};
}

/* The tile that workgroup `turn` of n_tiles * row_tiles takes.  Workgroups go to the eight
 * XCDs in turn: each XCD has a stretch of the tiles, in groups of 8 row tiles that share
 * what its L2 holds of W.  The host knows the experts' tiles only at most: row_tiles are
 * those that there are (else the last XCDs have none, 1190 us instead of 1110 for 8
 * experts of 1000 rows). */
__device__ static inline void f8_turn(int turn, int n_tiles, int row_tiles, int &row_tile, int &n_tile)
{
	const int all = n_tiles * row_tiles, xcd = turn % 8;
	const int id = xcd * (all / 8) + (xcd < all % 8 ? xcd : all % 8) + turn / 8;
	const int group = id / (8 * n_tiles), g0 = group * 8;
	const int many = row_tiles - g0 < 8 ? row_tiles - g0 : 8;
	const int in = id - group * 8 * n_tiles;
	row_tile = g0 + in % many;
	n_tile = in / many;
}

/* silu(a) * b.  16-bit outputs take the exponential and the reciprocal as the hardware
 * has them, 2^-22 and |a| 2^-24 off in relation, far inside their rounding (the others'
 * instructions for 64 outputs a lane took 4 us of each tile's 60).  0 where silu(a) is below
 * 2^-119: the reciprocal of more than 2^126 is, and in fp32 the exponential's infinity's. */
template <int TY> __device__ static inline float f8_gate(float a, float b)
{
	if constexpr (TY == HIP_F8_F32)
		return a / (1.0f + expf(-a)) * b;
	return a * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * a)) * b;
}

/*
 * A wave's outputs of 16 rows from r0 on, 4 N neighbouring ones of each from n0 on: lane l
 * has N of row l % 16 from N (l / 16) on.  They change lanes first, so that four lanes
 * next to each other have a row's 4 N: stores of lanes 16 apart are not joined to the 64
 * bytes that they make (112 us instead of 103, 8192 x 8192 x 1024).
 */
template <int TY, bool GATED, int N>
__device__ static inline void f8_store(const f8_mul_args &A, const f8_rows_of &R, int r0, int n0, float *y)
{
	typedef kv_type<TY> T;
	typedef kv_vec<TY, N> vec;
	constexpr int WORDS = sizeof(vec) / 4;
	union {
		vec v;
		u32 w[WORDS];
	} o;
	const int lane = f8_lane();
	if (!GATED && A.add) {
		const int r = r0 + lane % 16, n = n0 + lane / 16 * N;
		const typename T::t *p = (const typename T::t *)A.add + r * A.add_stride + n;
		if (r < R.b && n + N <= A.n) {
			const vec v = *(const vec *)p;
#pragma unroll
			for (int u = 0; u < N; u++)
				y[u] += T::get(v.v[u]);
		} else if (r < R.b) {
#pragma unroll
			for (int u = 0; u < N; u++)
				if (n + u < A.n)
					y[u] += T::get(p[u]);
		}
	}
#pragma unroll
	for (int u = 0; u < N; u++)
		o.v.v[u] = T::put(y[u]);
	const int turned = (lane % 4 * 16 + lane / 4) * 4;
#pragma unroll
	for (int w = 0; w < WORDS; w++)
		o.w[w] = __builtin_amdgcn_ds_bpermute(turned, o.w[w]);
	const int r = r0 + lane / 4, n = n0 + lane % 4 * N;
	if (r >= R.b)
		return;
	typename T::t *q = (typename T::t *)A.out + r * A.out_stride + n;
	if (n + N <= A.n) {
		*(vec *)q = o.v;
	} else {
#pragma unroll
		for (int u = 0; u < N; u++)
			if (n + u < A.n)
				q[u] = o.v.v[u];
	}
}

/* 16 bytes a lane from its address to lds + 16 * lane, in flight until a wait that the
 * caller makes (moe_device.h's dma_dwordx4 with whole addresses) */
__device__ static inline void f8_dma16(const uint8_t *p, u32 lds)
{
	asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
		     :
		     : "v"(p), "{m0}"(__builtin_amdgcn_readfirstlane(lds))
		     : "memory");
}

/* An address that all lanes share, for scalar registers */
__device__ static inline uint64_t f8_shared(const uint8_t *p)
{
	const uint64_t b = (uint64_t)(uintptr_t)p;
	return (uint64_t)(u32)__builtin_amdgcn_readfirstlane((int)(u32)b) |
	       ((uint64_t)(u32)__builtin_amdgcn_readfirstlane((int)(u32)(b >> 32)) << 32);
}

/* The first form from such a base.  The compiler may bring it to its scalar registers
 * right before, by vector instructions, and does not know that these five wait states
 * are needed then. */
__device__ static inline void f8_dma16(uint64_t base, u32 off, u32 lds)
{
	asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1"
		     :
		     : "v"(off), "s"(base), "{m0}"(__builtin_amdgcn_readfirstlane(lds))
		     : "memory");
}

/* The first form, 4 bytes a lane */
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

/* The row of X that row i of a tile comes from (a tile's last row past its rows; from[r]
 * is row r's); what is outside X reads its first row, and its outputs become NaN */
__device__ static inline int f8_source(const f8_mul_args &A, const f8_rows_of &R, const int *from, int i)
{
	const int r = R.a + i < R.b ? R.a + i : R.b - 1;
	const int x = A.from ? from[r] : r;
	return (unsigned)x < (unsigned)A.x_rows ? x : 0;
}

/* Where a lane's scale of slot `slot` of a tile starts, and how far the next block's is:
 * X's rows 64 a slot, then W's, one for each of WN x NR outputs and M matrices */
template <int M, int NR, int WN>
__device__ static inline void f8_scale_from(const f8_mul_args &A, const f8_rows_of &R, const int *from,
					    int n0, int slot, int x_slots, const float *&p, long &step)
{
	const int lane = f8_lane();
	if (slot < x_slots) {
		p = A.xs + f8_source(A, R, from, slot * 64 + lane);
		step = A.xs_stride;
	} else {
		const int m = lane % M;
		int n = n0 + lane / M % WN * NR;
		n = n < A.n ? n : A.n - 1;
		p = A.ws[m] + R.e * A.ws_step[m] + n / HIP_F8_BLOCK * A.ws_stride[m];
		step = 1;
	}
}

/* A wave's sums, of rows r0 .. and outputs n0 .., gated and stored: EACH operands give
 * a lane neighbouring outputs; from[r] is row r's of X */
template <int TY, bool GATED, int NA, int NB, int EACH>
__device__ static inline void f8_finish(const f8_mul_args &A, const f8_rows_of &R, const int *from, int r0,
					int n0, const float (&acc)[NA][NB][4])
{
	constexpr int FA = GATED ? NA / 2 : NA;
	const int lane = f8_lane();
#pragma unroll
	for (int b = 0; b < NB; b++) {
		const int r = r0 + b * 16 + lane % 16;
		const bool bad = A.from && r < R.b && (unsigned)from[r] >= (unsigned)A.x_rows;
#pragma unroll
		for (int f = 0; f < FA; f += EACH) {
			float out[4 * EACH];
#pragma unroll
			for (int i = 0; i < 4 * EACH; i++) {
				const float v = acc[f + i / 4][b][i % 4];
				out[i] = GATED ? f8_gate<TY>(v, acc[NA - FA + f + i / 4][b][i % 4]) : v;
				if (bad)
					out[i] = __builtin_nanf("");
			}
			f8_store<TY, GATED, 4 * EACH>(A, R, r0 + b * 16, n0 + f * 16, out);
		}
	}
}

/*
 * Tiles of 16 NB WT rows of X and 16 NA WN rows of W (gated: half of them W's, half
 * up's), a wave 16 NB by 16 NA of them.  A step is a block of 128 channels, in two
 * parts: X's rows with their scales and half of W's operands, then the other half.
 * Each part has STAGES buffers, filled by loads that go past the registers.  A part's
 * buffer is free, and is filled for STAGES steps later, once all waves have read it,
 * which they do an operand ahead of its products: a load has STAGES - 1/2 steps to
 * arrive, and the reads after a meeting have an operand's products to hide behind.
 *
 * The order of the instructions is this source's (sched_barrier): a product, then the
 * scaling of the one LAG before it, four instructions that the matrix cores' 32 cycles
 * cover.  Left to itself the compiler kept fewer sums and waited for each (989 us
 * instead of 925, 8192 rows by 28672 x 4096 gated).
 *
 * STREAM: a workgroup a compute unit takes tile after tile, gridDim.x apart, and its loads
 * go on over the border: a tile's last steps ask for the next one's first blocks, which arrive
 * while its outputs are stored.  Where the next tile is, and from which rows it comes, is
 * found in LDS, a step after the tile's start (98 -> 95 us, 8192 rows by 8192 x 1024
 * gated; two small workgroups a unit cover each other's borders by themselves).
 *
 * 8192 rows by 28672 x 4096 gated, bf16: 868 to 905 us, 2120 to 2220 TFLOP/s, of the
 * 2600 that a library's product of codes alone reaches; the matrix cores work in 51 % of
 * the cycles, at 1.9 to 2 GHz, which is what the power allows: without any loads
 * 2500 to 2900, products and scalings of registers alone 3600 (4400 with all data the same).
 *
 * A row's 128 bytes are eight pieces of 16; piece p lies at place p ^ (row % 8), so
 * that the 16 rows whose same piece an operand's read takes meet no bank twice.  Row
 * i of an operand's 16 is the output that gives a lane 16 bytes of neighbouring ones
 * from as many operands as that takes, and four lanes 64 bytes.
 */
template <int TY, bool GATED, int NA, int NB, int WN, int WT, int STAGES, bool STREAM>
__global__ __launch_bounds__(64 * WN * WT) void k_f8_tile(f8_mul_args A, int n_tiles, int row_tiles)
{
	constexpr int M = GATED ? 2 : 1, FA = NA / M; /* operands of one matrix */
	constexpr int BN = 16 * NA * WN, BT = 16 * NB * WT, NO = BN / M, HALF = NA / 2;
	constexpr int NW = WN * WT, SCALES = BT < 64 ? 64 : BT;
	constexpr int ROWS1 = BT + BN / 2, ROWS2 = BN / 2;
	constexpr int XSLOTS = BT / 8 / NW, SLOTS1 = ROWS1 / 8 / NW, SLOTS2 = ROWS2 / 8 / NW;
	constexpr int BYTES1 = ROWS1 * HIP_F8_BLOCK + SCALES * 4 + 256, BYTES2 = ROWS2 * HIP_F8_BLOCK;
	constexpr int AHEAD = (STAGES - 1) * (SLOTS1 + 1 + SLOTS2); /* loads that a wait leaves in flight */
	constexpr int LAG = NB < 3 ? NB : 3; /* sums that are not scaled yet */
	constexpr int EACH = TY == HIP_F8_F32 || FA == 1 ? 1 : 2; /* operands whose outputs neighbour */
	static_assert(BT / 8 % NW == 0 && ROWS2 / 8 % NW == 0, "whole loads");
	static_assert(NA % 2 == 0 && HIP_F8_BLOCK % (16 * FA) == 0 && FA % EACH == 0, "two parts, one scale");
	static_assert(NA * NB % 4 == 0, "the sums' places go round with the steps");
	static_assert(SCALES / 64 < NW && WN * M <= 64, "a wave is left for W's scales");
	typedef f8_operand<TY == HIP_F8_F32> operand;
	__shared__ __attribute__((aligned(16))) uint8_t lds[STAGES * (BYTES1 + BYTES2)];
	__shared__ int starts[STREAM ? F8_MAX_COUNT + 1 : 1], froms[STREAM ? 2 : 1][STREAM ? BT : 1];

	const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
	const int wn = wave % WN, wt = wave / WN;
	/* what a stream asks about experts and rows for its next tiles comes from LDS: a load
	 * into registers would wait for all that are in flight */
	if constexpr (STREAM) {
		if (A.start) {
			for (int i = threadIdx.x; i <= A.count; i += 64 * NW)
				starts[i] = A.start[i];
			__syncthreads();
		}
	}
	const int *const start = STREAM ? starts : A.start;
	row_tiles = f8_row_tiles<BT>(A, start, row_tiles);
	const int turns = n_tiles * row_tiles;
	int turn = blockIdx.x;
	if (turn >= turns)
		return;
	auto take = [&](int at, f8_rows_of &T, int &tn) {
		int tile;
		f8_turn(at, n_tiles, row_tiles, tile, tn);
		tn *= NO;
		T = f8_find<BT>(A, start, tile);
	};
	f8_rows_of R, next_R = {0, 0, 0};
	int n0, next_n0 = 0, ring = 0;
	bool more = false;
	take(turn, R, n0);
	if constexpr (STREAM) {
		if (A.from) {
			for (int i = threadIdx.x; i < BT; i += 64 * NW)
				froms[0][i] = A.from[R.a + i < R.b ? R.a + i : R.b - 1];
			__syncthreads();
		}
	}
	/* its rows' sources, from[r] for row r */
	auto from_of = [&](const f8_rows_of &T, int which) -> const int * {
		return STREAM ? froms[which] - T.a : A.from;
	};

	/* what this wave loads of a tile: slots of eight rows, X's, W's first half, W's second; a
	 * row by its distance from the tile's first, or where X is gathered from X's first (32
	 * bits; not in a stream X's whole addresses) */
	const int piece = ((lane % 8) ^ (lane / 8)) * 16, last = (A.k - 1) & ~15;
	uint64_t from_x = 0, from_w, from_u;
	u32 off[SLOTS1 + SLOTS2];
	const uint8_t *far[STREAM ? 1 : XSLOTS];
	/* and of the scales: X's 64 at a time, then W's */
	const float *ps;
	long ps_step;
	const int sslot = wave < SCALES / 64 ? wave : SCALES / 64;
	auto w_row = [&](int i, int tn) {
		/* half (gated: matrix), wn, operand of the half, row of it */
		const int j = (wave + i * NW) * 8 + f8_lane() / 8 - BT, r = j % 16;
		const int f = (j / (BN / 2) * HALF + j / 16 % HALF) % FA;
		const int n = j / (16 * HALF) % WN * (16 * FA) + f / EACH * (16 * EACH) +
			      r / 4 * (4 * EACH) + f % EACH * 4 + r % 4;
		return (u32)(tn + n < A.n ? n : A.n - 1 - tn);
	};
	auto set1 = [&](const f8_rows_of &T, int tn, const int *from) {
		if constexpr (STREAM)
			from_x = f8_shared(A.from ? A.x : A.x + T.a * A.x_stride);
		from_w = f8_shared(A.w[0] + T.e * A.w_step[0] + tn * A.w_stride[0]);
#pragma unroll
		for (int i = 0; i < SLOTS1; i++) {
			if (i >= XSLOTS) {
				off[i] = w_row(i, tn) * (u32)A.w_stride[0];
				continue;
			}
			const int x = f8_source(A, T, from, (wave + i * NW) * 8 + f8_lane() / 8);
			if constexpr (STREAM)
				off[i] = (u32)(A.from ? x : x - T.a) * (u32)A.x_stride;
			else
				far[i] = A.x + x * A.x_stride;
		}
		f8_scale_from<M, 16 * FA, WN>(A, T, from, tn, sslot, SCALES / 64, ps, ps_step);
	};
	auto set2 = [&](const f8_rows_of &T, int tn) {
		from_u = f8_shared(A.w[M - 1] + T.e * A.w_step[M - 1] + tn * A.w_stride[M - 1]);
#pragma unroll
		for (int i = SLOTS1; i < SLOTS1 + SLOTS2; i++)
			off[i] = w_row(i, tn) * (u32)A.w_stride[M - 1];
	};
	set1(R, n0, from_of(R, 0));
	set2(R, n0);
	const int blocks = (A.k + HIP_F8_BLOCK - 1) / HIP_F8_BLOCK;
	const bool rest = A.k % HIP_F8_BLOCK;
	uint8_t *const lds2 = lds + STAGES * BYTES1;
	const u32 base1 = lds_addr(lds), base2 = lds_addr(lds2);
	/* a block's part into a buffer; past the last block the next tile's, or without one the
	 * last again, which nothing reads */
	auto load1 = [&](int kb, int stage) {
		kb = kb < blocks ? kb : STREAM && more ? kb - blocks : blocks - 1;
		int c = kb * HIP_F8_BLOCK + piece;
		c = c < last ? c : last; /* nothing past the row's last 16 that hold any is read */
#pragma unroll
		for (int i = 0; i < SLOTS1; i++) {
			const u32 to = base1 + stage * BYTES1 + (wave + i * NW) * 1024;
			if (!STREAM && i < XSLOTS)
				f8_dma16(far[STREAM ? 0 : i < XSLOTS ? i : 0] + c, to);
			else
				f8_dma16(i < XSLOTS ? from_x : from_w, off[i] + c, to);
		}
		f8_dma4(ps + kb * ps_step, base1 + stage * BYTES1 + ROWS1 * HIP_F8_BLOCK + sslot * 256);
	};
	auto load2 = [&](int kb, int stage) {
		kb = kb < blocks ? kb : STREAM && more ? kb - blocks : blocks - 1;
		int c = kb * HIP_F8_BLOCK + piece;
		c = c < last ? c : last;
#pragma unroll
		for (int i = 0; i < SLOTS2; i++)
			f8_dma16(from_u, off[SLOTS1 + i] + c, base2 + stage * BYTES2 + (wave + i * NW) * 1024);
	};
	/* zeros behind the last block's channels; rows is a multiple of eight */
	auto cut = [&](uint8_t *buf, int rows) {
		for (int i = threadIdx.x; i < rows * 8; i += 64 * NW) {
			const int c = (blocks - 1) * HIP_F8_BLOCK + ((i % 8) ^ (i / 8 % 8)) * 16;
			i32x4 *q = (i32x4 *)(buf + i * 16);
			if (c + 16 > A.k)
				*q = f8_masked(*q, c, A.k);
		}
		f8_meet<63>();
	};

	const int place = ((lane / 16) ^ (lane % 8)) * 16;
	const int xo = (wt * 16 * NB + lane % 16) * HIP_F8_BLOCK + place;
	const int wo = (wn * 16 * HALF + lane % 16) * HIP_F8_BLOCK + place;
	f8_raw xr[NB], wr[2];
	float s[M][NB], s_last[LAG] = {};
	auto read_x = [&](int stage, int b) { xr[b].get(lds + stage * BYTES1 + xo + b * 2048, place); };
	auto read_w = [&](int stage, int a) {
		const uint8_t *w = a < HALF ? lds + stage * BYTES1 + BT * HIP_F8_BLOCK : lds2 + stage * BYTES2;
		wr[a % 2].get(w + wo + a % HALF * 2048, place);
	};
	auto read_s = [&](int stage) {
		const float *sx = (const float *)(lds + stage * BYTES1 + ROWS1 * HIP_F8_BLOCK);
#pragma unroll
		for (int b = 0; b < NB; b++)
#pragma unroll
			for (int m = 0; m < M; m++)
				s[m][b] = sx[(wt * NB + b) * 16 + lane % 16] * sx[SCALES + wn * M + m];
	};

#pragma unroll
	for (int i = 0; i < STAGES; i++) {
		load1(i, i);
		if (i + 1 < STAGES)
			load2(i, i);
	}
	f8_meet<AHEAD>();
	load2(STAGES - 1, STAGES - 1);
	if (blocks == 1 && rest)
		cut(lds, ROWS1);
	read_w(0, 0);
#pragma unroll
	for (int b = 0; b < NB; b++)
		read_x(0, b);
	read_s(0);

	float acc[NA][NB][4] = {};
	floatx4 y[4] = {};
	int stage = 0;
	for (int kb = 0;;) {
		const int next = stage + 1 == STAGES ? 0 : stage + 1;
		operand x[NB], w;
#pragma unroll
		for (int b = 0; b < NB; b++)
			x[b].set(xr[b]);
#pragma unroll
		for (int a = 0; a < NA; a++) {
			if (a == HALF - 1) { /* all have read the first part */
				f8_meet<AHEAD>();
				if (STREAM && kb == 0) {
					more = turn + (int)gridDim.x < turns;
					if (more) {
						take(turn + gridDim.x, next_R, next_n0);
						if (A.from) { /* read two meetings on */
							const int i = wave % (BT / 64) * 64 + f8_lane();
							const int r = next_R.a + i < next_R.b ? next_R.a + i : next_R.b - 1;
							f8_dma4((const float *)(A.from + r),
								lds_addr(&froms[STREAM ? ring ^ 1 : 0][wave % (BT / 64) * 64]));
						}
					}
				}
				if (STREAM && kb == blocks - STAGES && more)
					set1(next_R, next_n0, from_of(next_R, ring ^ 1));
				load1(kb + STAGES, stage);
				if (kb == blocks - 1 && rest)
					cut(lds2 + stage * BYTES2, ROWS2);
			}
			if (a == NA - 1) { /* all have read the second */
				f8_meet<AHEAD>();
				if (STREAM && kb == blocks - STAGES && more)
					set2(next_R, next_n0);
				load2(kb + STAGES, stage);
				if (kb == blocks - 2 && rest)
					cut(lds + next * BYTES1, ROWS1);
			}
			w.set(wr[a % 2]);
			if (a < NA - 1)
				read_w(stage, a + 1);
			else
				read_w(next, 0);
			__builtin_amdgcn_sched_barrier(0);
#pragma unroll
			for (int b = 0; b < NB; b++) {
				const int i = a * NB + b, j = (i + NA * NB - LAG) % (NA * NB);
				y[i % 4] = operand::mul(w, x[b]);
				if (a == NA - 1)
					read_x(next, b);
				const float f = i < LAG ? s_last[i] : s[j / NB / FA][j % NB];
#pragma unroll
				for (int u = 0; u < 4; u++) {
					acc[j / NB][j % NB][u] = __builtin_fmaf(y[j % 4][u], f, acc[j / NB][j % NB][u]);
					asm volatile("" : "+v"(acc[j / NB][j % NB][u])); /* here, not behind a branch */
				}
				__builtin_amdgcn_sched_barrier(0);
			}
		}
#pragma unroll
		for (int i = 0; i < LAG; i++)
			s_last[i] = s[M - 1][NB - LAG + i];
		read_s(next);
		stage = next;
		if (++kb < blocks)
			continue;
#pragma unroll
		for (int i = 0; i < LAG; i++)
#pragma unroll
			for (int u = 0; u < 4; u++)
				acc[NA - 1][NB - LAG + i][u] = __builtin_fmaf(y[(NA * NB - LAG + i) % 4][u], s_last[i],
									      acc[NA - 1][NB - LAG + i][u]);
		if (!more)
			f8_meet<0>(); /* no load outlives the workgroup's LDS */
		f8_finish<TY, GATED, NA, NB, EACH>(A, R, from_of(R, ring), R.a + wt * NB * 16, n0 + wn * 16 * FA, acc);
		if (!more)
			break;
		turn += gridDim.x;
		R = next_R;
		n0 = next_n0;
		ring ^= 1;
		kb = 0;
#pragma unroll
		for (int a = 0; a < NA; a++)
#pragma unroll
			for (int b = 0; b < NB; b++)
#pragma unroll
				for (int u = 0; u < 4; u++)
					acc[a][b][u] = 0.0f;
#pragma unroll
		for (int i = 0; i < LAG; i++) {
			s_last[i] = 0.0f;
			y[(NA * NB - LAG + i) % 4] = floatx4{0, 0, 0, 0};
		}
	}
}

/*
 * Tiles of 16 NB WT rows of X and 16 NA WN rows of W (gated: half of them W's, half
 * up's) where there are few of them: KS groups of WN WT waves take the blocks of
 * channels in turn, each into LDS of its own, and add their sums up at the end.  All
 * groups meet once a step, so that a step's waits are paid once for KS blocks (333 rows
 * by 4096 x 4096, f16: 17.3 us, four of them the call's).  Rows lie in LDS and outputs in the
 * lanes as in k_f8_tile.
 */
template <int TY, bool GATED, int NA, int NB, int WN, int WT, int KS, int STAGES>
__global__ __launch_bounds__(64 * WN * WT * KS) void k_f8_mid(f8_mul_args A, int n_tiles, int row_tiles)
{
	constexpr int M = GATED ? 2 : 1, FA = NA / M;
	constexpr int BN = 16 * NA * WN, BT = 16 * NB * WT, NO = BN / M, NW = WN * WT;
	constexpr int XSLOTS = BT / 8 / NW, SLOTS = (BN + BT) / 8 / NW, SCALES = BT < 64 ? 64 : BT;
	constexpr int BYTES = (BN + BT) * HIP_F8_BLOCK + SCALES * 4 + 256; /* of a block */
	constexpr int EACH = TY == HIP_F8_F32 || FA == 1 ? 1 : 2;
	static_assert(BT / 8 % NW == 0 && BN / 8 % NW == 0, "whole loads");
	static_assert(NA % M == 0 && HIP_F8_BLOCK % (16 * FA) == 0 && FA % EACH == 0, "one scale");
	static_assert(SCALES / 64 < NW && WN * M <= 64, "a wave is left for W's scales");
	static_assert((KS - 1) * BN * BT * 4 <= STAGES * KS * BYTES, "the groups' sums");
	typedef f8_operand<TY == HIP_F8_F32> operand;
	__shared__ __attribute__((aligned(16))) uint8_t lds[STAGES * KS * BYTES];

	const int lane = threadIdx.x % 64;
	const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64 % NW);
	const int ks = __builtin_amdgcn_readfirstlane(threadIdx.x / 64 / NW);
	const int wn = wave % WN, wt = wave / WN;
	row_tiles = f8_row_tiles<BT>(A, A.start, row_tiles);
	if ((int)blockIdx.x >= n_tiles * row_tiles)
		return;
	int tile, n0;
	f8_turn(blockIdx.x, n_tiles, row_tiles, tile, n0);
	n0 *= NO;
	const f8_rows_of R = f8_find<BT>(A, A.start, tile);

	const int piece = ((lane % 8) ^ (lane / 8)) * 16, last = (A.k - 1) & ~15;
	const uint8_t *p[SLOTS];
#pragma unroll
	for (int i = 0; i < SLOTS; i++) {
		const int row = (wave + i * NW) * 8 + lane / 8;
		if (i < XSLOTS) {
			p[i] = A.x + f8_source(A, R, A.from, row) * A.x_stride;
		} else {
			/* wn, operand of its NA, row of it */
			const int j = row - BT, r = j % 16, a = j / 16 % NA, m = a / FA, f = a % FA;
			int n = n0 + j / (16 * NA) * (16 * FA) + f / EACH * (16 * EACH) + r / 4 * (4 * EACH) +
				f % EACH * 4 + r % 4;
			n = n < A.n ? n : A.n - 1;
			p[i] = m ? A.w[M - 1] + R.e * A.w_step[M - 1] + n * A.w_stride[M - 1]
				 : A.w[0] + R.e * A.w_step[0] + n * A.w_stride[0];
		}
	}
	const float *ps;
	long ps_step;
	const int sslot = wave < SCALES / 64 ? wave : SCALES / 64;
	f8_scale_from<M, 16 * FA, WN>(A, R, A.from, n0, sslot, SCALES / 64, ps, ps_step);

	const int blocks = (A.k + HIP_F8_BLOCK - 1) / HIP_F8_BLOCK, steps = (blocks + KS - 1) / KS;
	const u32 base = lds_addr(lds);
	auto load = [&](int step, int stage) {
		int kb = step * KS + ks;
		kb = kb < blocks ? kb : blocks - 1;
		int c = kb * HIP_F8_BLOCK + piece;
		c = c < last ? c : last;
		const u32 to = base + (stage * KS + ks) * BYTES;
#pragma unroll
		for (int i = 0; i < SLOTS; i++)
			f8_dma16(p[i] + c, to + (wave + i * NW) * 1024);
		f8_dma4(ps + kb * ps_step, to + (BN + BT) * HIP_F8_BLOCK + sslot * 256);
	};
	const int place = ((lane / 16) ^ (lane % 8)) * 16;
	const int xo = (wt * 16 * NB + lane % 16) * HIP_F8_BLOCK + place;
	const int wo = (BT + wn * 16 * NA + lane % 16) * HIP_F8_BLOCK + place;
	float acc[NA][NB][4] = {};
#pragma unroll
	for (int i = 0; i < STAGES - 1; i++)
		load(i, i);
	int stage = 0;
	for (int step = 0; step < steps; step++) {
		f8_meet<(STAGES - 2) * (SLOTS + 1)>();
		load(step + STAGES - 1, stage == 0 ? STAGES - 1 : stage - 1);
		uint8_t *buf = lds + (stage * KS + ks) * BYTES;
		const int kb = step * KS + ks;
		if (step == steps - 1 && A.k % HIP_F8_BLOCK) {
			if (kb == blocks - 1)
				for (int i = wave * 64 + lane; i < (BN + BT) * 8; i += 64 * NW) {
					const int c = kb * HIP_F8_BLOCK + ((i % 8) ^ (i / 8 % 8)) * 16;
					i32x4 *q = (i32x4 *)(buf + i * 16);
					if (c + 16 > A.k)
						*q = f8_masked(*q, c, A.k);
				}
			f8_meet<63>();
		}
		if (kb < blocks) {
			const float *sx = (const float *)(buf + (BN + BT) * HIP_F8_BLOCK);
			f8_raw xr[NB], wr[2];
			float s[M][NB];
			wr[0].get(buf + wo, place);
#pragma unroll
			for (int b = 0; b < NB; b++)
				xr[b].get(buf + xo + b * 2048, place);
#pragma unroll
			for (int b = 0; b < NB; b++)
#pragma unroll
				for (int m = 0; m < M; m++)
					s[m][b] = sx[(wt * NB + b) * 16 + lane % 16] * sx[SCALES + wn * M + m];
			operand x[NB];
#pragma unroll
			for (int b = 0; b < NB; b++)
				x[b].set(xr[b]);
			floatx4 y[2][NB];
#pragma unroll
			for (int a = 0; a <= NA; a++) {
				operand w;
				if (a < NA)
					w.set(wr[a % 2]);
				if (a + 1 < NA)
					wr[(a + 1) % 2].get(buf + wo + (a + 1) * 2048, place);
#pragma unroll
				for (int b = 0; b < NB; b++) {
					if (a < NA)
						y[a % 2][b] = operand::mul(w, x[b]);
					if (a > 0)
#pragma unroll
						for (int u = 0; u < 4; u++)
							acc[a - 1][b][u] = __builtin_fmaf(y[(a - 1) % 2][b][u],
											  s[(a - 1) / FA][b], acc[a - 1][b][u]);
				}
			}
		}
		stage = stage + 1 == STAGES ? 0 : stage + 1;
	}
	f8_meet<0>(); /* no load outlives the workgroup's LDS */
	floatx4 *sums = (floatx4 *)lds; /* [ks - 1][wave][a][b][lane] */
	if (KS > 1) {
		if (ks > 0)
#pragma unroll
			for (int a = 0; a < NA; a++)
#pragma unroll
				for (int b = 0; b < NB; b++)
					sums[((((ks - 1) * NW + wave) * NA + a) * NB + b) * 64 + lane] =
						floatx4{acc[a][b][0], acc[a][b][1], acc[a][b][2], acc[a][b][3]};
		__syncthreads();
		if (ks > 0)
			return;
#pragma unroll
		for (int g = 0; g < KS - 1; g++)
#pragma unroll
			for (int a = 0; a < NA; a++)
#pragma unroll
				for (int b = 0; b < NB; b++) {
					const floatx4 v = sums[(((g * NW + wave) * NA + a) * NB + b) * 64 + lane];
#pragma unroll
					for (int u = 0; u < 4; u++)
						acc[a][b][u] += v[u];
				}
	}
	f8_finish<TY, GATED, NA, NB, EACH>(A, R, A.from, R.a + wt * NB * 16, n0 + wn * 16 * FA, acc);
}

/*
 * Few rows: 16 NT rows of X and 16 NF outputs a workgroup, whose NW waves take the
 * blocks of channels in turn, each with loads of its own from W and X, DEPTH blocks
 * ahead, and no LDS but for the waves' sums at the end.  W is read as its rows lie,
 * 64 bytes of each a load; what bounds it is how much of W is in flight.  16 rows in 8
 * experts of 28672 x 4096 gated: 170 us, 5.5 TB/s; a row by 50304 x 2048, fp32: 18 us, 5.7 TB/s.
 */
template <int TY, bool GATED, int NF, int NT, int NW, int DEPTH>
__global__ __launch_bounds__(64 * NW) void k_f8_few(f8_mul_args A, int n_tiles, int)
{
	constexpr int M = GATED ? 2 : 1, FN = NF * M;
	typedef f8_operand<TY == HIP_F8_F32> operand;
	__shared__ floatx4 sums[NW][FN][NT][64];
	const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
	const int tile = blockIdx.x / n_tiles, n0 = blockIdx.x % n_tiles * (16 * NF);
	const f8_rows_of R = f8_find<16 * NT>(A, A.start, tile);
	if (R.a >= R.b)
		return;
	const int piece = lane / 16 * 16, last = (A.k - 1) & ~15; /* of each 64 channels */
	const uint8_t *px[NT], *pw[FN];
	const float *sx[NT], *sw[M];
#pragma unroll
	for (int t = 0; t < NT; t++) {
		int x = R.a + t * 16 + lane % 16;
		x = x < R.b ? x : R.b - 1;
		x = A.from ? A.from[x] : x;
		x = (unsigned)x < (unsigned)A.x_rows ? x : 0;
		px[t] = A.x + x * A.x_stride;
		sx[t] = A.xs + x;
	}
#pragma unroll
	for (int f = 0; f < FN; f++) {
		const int m = f / NF, n = n0 + f % NF * 16 + lane % 16;
		pw[f] = A.w[m] + R.e * A.w_step[m] + (n < A.n ? n : A.n - 1) * A.w_stride[m];
	}
#pragma unroll
	for (int m = 0; m < M; m++)
		sw[m] = A.ws[m] + R.e * A.ws_step[m] + n0 / HIP_F8_BLOCK * A.ws_stride[m];
	const int blocks = (A.k + HIP_F8_BLOCK - 1) / HIP_F8_BLOCK;

	struct {
		f8_raw x[NT], w[FN];
		float sx[NT], sw[M];
	} in[DEPTH + 1];
	auto load = [&](int kb, int i) {
		const int c = kb * HIP_F8_BLOCK + piece;
		const int lo = c < last ? c : last, hi = c + 64 < last ? c + 64 : last;
#pragma unroll
		for (int f = 0; f < FN; f++)
			in[i].w[f].get2(pw[f] + lo, pw[f] + hi);
#pragma unroll
		for (int t = 0; t < NT; t++) {
			in[i].x[t].get2(px[t] + lo, px[t] + hi);
			in[i].sx[t] = sx[t][kb * A.xs_stride];
		}
#pragma unroll
		for (int m = 0; m < M; m++)
			in[i].sw[m] = sw[m][kb];
	};
	floatx4 acc[FN][NT] = {};
	auto use = [&](int kb, int i) {
		if ((kb + 1) * HIP_F8_BLOCK > A.k) {
			const int c = kb * HIP_F8_BLOCK + piece;
#pragma unroll
			for (int f = 0; f < FN; f++)
				in[i].w[f].cut(c, A.k);
#pragma unroll
			for (int t = 0; t < NT; t++)
				in[i].x[t].cut(c, A.k);
		}
		operand w[FN];
#pragma unroll
		for (int f = 0; f < FN; f++)
			w[f].set(in[i].w[f]);
#pragma unroll
		for (int t = 0; t < NT; t++) {
			operand x;
			x.set(in[i].x[t]);
#pragma unroll
			for (int f = 0; f < FN; f++) {
				const floatx4 y = operand::mul(w[f], x);
				const float s = in[i].sx[t] * in[i].sw[f / NF];
#pragma unroll
				for (int u = 0; u < 4; u++)
					acc[f][t][u] = __builtin_fmaf(y[u], s, acc[f][t][u]);
			}
		}
	};
#pragma unroll
	for (int i = 0; i < DEPTH; i++)
		if (wave + i * NW < blocks)
			load(wave + i * NW, i);
	for (int kb = wave; kb < blocks; kb += (DEPTH + 1) * NW) {
#pragma unroll
		for (int i = 0; i <= DEPTH; i++) {
			const int at = kb + i * NW, ahead = at + DEPTH * NW;
			if (ahead < blocks)
				load(ahead, (i + DEPTH) % (DEPTH + 1));
			if (at < blocks)
				use(at, i);
		}
	}
#pragma unroll
	for (int f = 0; f < FN; f++)
#pragma unroll
		for (int t = 0; t < NT; t++)
			sums[wave][f][t][lane] = acc[f][t];
	__syncthreads();
	for (int i = wave; i < NF * NT; i += NW) {
		const int f = i % NF, t = i / NF, r = R.a + t * 16 + lane % 16;
		floatx4 y[M] = {};
#pragma unroll
		for (int m = 0; m < M; m++)
#pragma unroll
			for (int w = 0; w < NW; w++)
				y[m] += sums[w][m * NF + f][t][lane];
		const bool bad = A.from && r < R.b && (unsigned)A.from[r] >= (unsigned)A.x_rows;
		float out[4];
#pragma unroll
		for (int u = 0; u < 4; u++) {
			out[u] = GATED ? f8_gate<TY>(y[0][u], y[M - 1][u]) : y[0][u];
			if (bad)
				out[u] = __builtin_nanf("");
		}
		f8_store<TY, GATED, 4>(A, R, R.a + t * 16, n0 + f * 16, out);
	}
}

/*
 * The forms, and what a call costs in each.  With `n` of a form's workgroups to each of
 * the 256 compute units, rounded up where they are few, a call takes
 *   fixed + block * blocks + (n - 1) (more_fixed + more_block * blocks)
 * microseconds and 5 that all forms share, blocks of 128 channels; the first of them alone on
 * its unit, later ones next to others.  The four are there to choose by: they were fitted
 * to 420 calls, dense and grouped (16 to 8192 rows, 1024 to 14336 outputs, 400 to 5120 channels,
 * up to 64 experts), timed in every form, of which those within twice the fastest counted.
 * The form with the smallest sum took 2 % longer than the fastest on average, 16 bits and fp32, and in
 * nine of ten calls at most 8 %, in these and in 240 others.  What a form takes far
 * from where it is chosen they do not say: dense calls of whole rounds, measured and (by the
 * formula, with the 5),
 *
 *   4096 channels, us by workgroups      256          512           1024          2048
 *   16 bits  MID   32 x 128, 2 groups   13.1 (13.6)   23.3 (30.4)   43.5 (63.9)   84.2 (131)
 *            MID   64 x 64, 4 groups    12.5 (13.8)   22.9 (27.4)   42.4 (54.7)   82.2 (109)
 *            MID   64 x 128, 2 groups   17.6 (16.4)   31.5 (39.8)   59.8 (86.4)    118 (180)
 *            TILE  64 x 128             24.4 (22.9)   31.4 (37.3)   56.4 (66.3)    105 (124)
 *            TILE 128 x 128             28.2 (24.5)   46.1 (48.6)   87.6 (96.9)    171 (193)
 *            TILE 256 x 256             74.5 (65.4)    141 (121)     287 (232)     554 (454)
 *   fp32     MID   32 x 128, 2 groups   17.8 (19.0)   32.9 (40.1)   63.3 (82.1)    124 (166)
 *            MID   64 x 64, 4 groups    17.0 (17.2)   29.8 (34.7)   56.6 (69.6)    111 (140)
 *            MID   64 x 128, 2 groups   25.4 (25.1)   47.5 (53.6)   92.7 (110)     180 (224)
 *            MID  128 x 128, 2 groups   39.2 (37.6)   77.3 (80.0)    152 (165)     296 (334)
 *            TILE  64 x 128             35.2 (29.0)   47.2 (50.8)   82.9 (94.4)    158 (181)
 *            TILE 128 x 128             53.7 (46.2)   76.6 (82.8)    145 (156)     281 (302)
 *
 * TILE 256 x 256 takes 63 to 64 for 128 to 192 workgroups: with all units at work the clock
 * falls.  By the rows of 4096 x 4096, 16 bits: 2304 rows 62.9 in it and 61.2 in TILE 128 x 128,
 * 2816 63.4 and 63.4, 3584 67.9 and 82.2, 4096 75.3 and 87.1, 5120 (its 320 workgroups are two
 * rounds) 122 and 110; it is taken in all of these.  Sizes alone would not do: calls of many
 * rounds cost the same as larger tiles' calls of few.
 *
 * TILE's 64 x 128 by four waves with two stages, three workgroups a compute unit: eight
 * waves with three stages, two workgroups, took 46.3 and 86.7 us for 768 and 1536 (fp32
 * 70.7 and 138: four operands to convert for 4 products instead of six for 8).
 *
 * One to a few rows are bound by W's way from HBM: FEW.  4096 x 4096 for one row takes
 * 7.4 us where a tile takes 21, 50304 x 2048 18 where it takes 26.  Waves of 16 outputs
 * and eight to a workgroup where the outputs alone do not fill the chip (15.5 us
 * instead of 21.5, 16 rows of 14336 to 4096), else four (18.1 instead of 23.7, the 50304),
 * and 32 outputs where the product is gated (169 instead of 176, 16 tokens in 8 experts of 14336 x 4096).
 * Their costs were fitted to 420 calls of up to 128 rows or 40 for an expert, W from HBM; a gated
 * call's blocks count twice.  Up to 16 rows (8 for an expert, and few workgroups) they
 * are taken unasked, 4 % behind the fastest of all forms on average.  Where experts have 8
 * rows on average some have many more, and with many experts workgroups of 16 rows are tens
 * of thousands: from there on TILE is taken where its cost is 10 % below (512 rows in 64 experts
 * of 2048 x 1024: 34 us instead of 50, 33 instead of 51 with a skewed router; 10240 fp32 rows in 1024 of
 * 512 x 512 gated: 296 instead of 637, 282 instead of 636).  FEW_LONG up to 128 rows where it costs no more than
 * 15 % below others (24 rows of 4096 x 4096: 10.6 instead of 15.2 us, 48 of 1024 x 4096: 8.7 instead of
 * 11.7).  In 843 calls of more than those 16 and 8 rows, even and skewed, 5 % behind the
 * fastest on average, in nine of ten at most 17 %.
 */
#define F8_FORMS(X)                                                                    \
	/*  form        kernel   16-bit fp32  NA NB WN WT KS STAGES STREAM */               \
	X(FEW_LONG, few, 1, 1, 1, 1, 8, 2)                                             \
	X(FEW_WIDE, few, 1, 1, 1, 1, 4, 3)                                             \
	X(FEW_GATED, few, 1, 1, 2, 1, 4, 2)                                            \
	X(FEW_32, few, 1, 1, 2, 2, 4, 1)                                               \
	X(MID_32, mid, 1, 1, 2, 2, 4, 1, 2, 3)                                         \
	X(MID_64, mid, 1, 1, 2, 4, 2, 1, 4, 2)                                         \
	X(MID_128, mid, 1, 1, 2, 4, 4, 1, 2, 3)                                        \
	X(MID_SQUARE, mid, 0, 1, 4, 4, 2, 2, 2, 2)                                     \
	X(TILE_64, tile, 1, 1, 4, 2, 2, 2, 2, false)                                   \
	X(TILE_128, tile, 1, 0, 4, 2, 2, 4, 2, false)                                  \
	X(TILE_128F, tile, 0, 1, 4, 4, 2, 2, 2, false)                                 \
	X(TILE_256, tile, 1, 0, 8, 4, 2, 4, 2, true)

#define F8_CUS 256

enum {
#define X(FORM, ...) FORM,
	F8_FORMS(X)
#undef X
	FORMS
};

/* tiles and costs, by type (16 bits, fp32) */
static const struct {
	int bt, bn, threads;
	struct {
		float fixed, block, more_fixed, more_block;
	} us[2];
} forms[FORMS] = {
	/* in F8_FORMS' order */
	{16, 16, 512, {{2.9f, .035f, .65f, .077f}, {2.9f, .041f, .82f, .062f}}},
	{16, 16, 256, {{0, .081f, .66f, .03f}, {0, .126f, .61f, .075f}}},
	{16, 32, 256, {{0, .114f, 1.11f, .084f}, {.46f, .113f, 1.49f, .102f}}},
	{32, 32, 256, {{0, .2f, 1.11f, .165f}, {.66f, .158f, 1.13f, .18f}}},
	{32, 128, 512, {{3.2f, .17f, 3.3f, .42f}, {2.5f, .36f, 4.4f, .52f}}},
	{64, 64, 512, {{4.6f, .13f, 5.f, .27f}, {2.9f, .29f, 5.f, .39f}}},
	{64, 128, 512, {{2.8f, .27f, 5.4f, .56f}, {2.2f, .56f, 6.7f, .68f}}},
	{128, 128, 512, {{}, {5.7f, .84f, 8.8f, 1.05f}}},
	{64, 128, 256, {{2.2f, .49f, 2.3f, .38f}, {2.6f, .67f, 2.9f, .59f}}},
	{128, 128, 512, {{1.9f, .55f, 4.3f, .62f}, {}}},
	{128, 128, 256, {{}, {6.6f, 1.08f, 4.6f, 1.f}}},
	{256, 256, 512, {{10.8f, 1.55f, 10.1f, 1.42f}, {}}},
};

/* tiles of rows and of outputs; a grouped call's rows may end in a tile that is not
 * full for every expert */
static size_t row_tiles_of(const f8_mul_args *a, size_t bt)
{
	const size_t rows = (size_t)a->rows, count = (size_t)a->count;
	return a->start ? rows / bt + (rows < count ? rows : count) : (rows + bt - 1) / bt;
}

static size_t n_tiles_of(const f8_mul_args *a, int form)
{
	/* the tiles' outputs are half of their rows of W where two matrices share them */
	const size_t bn = (size_t)forms[form].bn / (form >= MID_32 && a->w[1] ? 2 : 1);
	return ((size_t)a->n + bn - 1) / bn;
}

static float cost_of(const f8_mul_args *a, int form, int fp32)
{
	const float bt = forms[form].bt, rows = a->rows, busy = rows < a->count ? rows : a->count;
	const bool few = form < MID_32;
	/* a workgroup's outputs are of one matrix (FEW: of both, which is twice the loads) */
	const float blocks = (a->k + HIP_F8_BLOCK - 1) / HIP_F8_BLOCK * (few && a->w[1] ? 2 : 1);
	float tiles = ceilf(rows / bt);
	if (a->start) {
		/* between experts that have the same rows and some whose last tile is half full */
		const float even = busy * ceilf(rows / busy / bt), uneven = rows / bt + .5f * busy;
		tiles = .5f * (even + (uneven > busy ? uneven : busy));
	}
	float n = tiles * n_tiles_of(a, form) / F8_CUS;
	n = n < 6 ? ceilf(n) : n;
	const float less = a->w[1] && !few ? .7f : 1; /* half the outputs to store */
	const auto &c = forms[form].us[fp32];
	return less * c.fixed + c.block * blocks + (n - 1) * (less * c.more_fixed + c.more_block * blocks);
}

void f8_mul_plan(const f8_mul_args *a, f8_plan *p)
{
	const size_t rows = (size_t)a->rows;
	const size_t per = a->start ? (rows + (size_t)a->count - 1) / (size_t)a->count : rows;
	const int fp32 = p->type == HIP_F8_F32;
	/* of few rows' forms the one that was measured there, or none; against others where there
	 * are enough workgroups that one of them may be much faster */
	int few = FORMS, first = MID_32;
	if (per <= (a->start ? 8 : 16)) {
		const size_t wide = row_tiles_of(a, 16) * (((size_t)a->n + 31) / 32);
		few = wide < 512 ? FEW_LONG : a->w[1] ? FEW_GATED : FEW_WIDE;
		first = a->start && wide >= 2048 ? TILE_64 : FORMS;
	} else if (a->start && per <= 24) {
		few = FEW_32;
		first = TILE_64;
	} else if (!a->start && per <= 128) {
		few = FEW_LONG;
	}
	float best = 0;
	if (few < FORMS) {
		p->form = few;
		best = cost_of(a, few, fp32) * (a->start ? .9f : 1.15f);
	}
	for (int f = first; f < FORMS; f++) {
		if (forms[f].us[fp32].block == 0)
			continue;
		/* its rows' distances from X's first are 32 bits; it asks for the next tile two
		 * steps ahead */
		if (f == TILE_256 &&
		    (a->k <= 2 * HIP_F8_BLOCK ||
		     (a->from && (size_t)a->x_rows * (size_t)a->x_stride >= ((size_t)1 << 32) - F8_MAX_K)))
			continue;
		const float us = cost_of(a, f, fp32);
		if (best == 0 || us < best) {
			best = us;
			p->form = f;
		}
	}
	p->threads = forms[p->form].threads;
	p->n_tiles = n_tiles_of(a, p->form);
	p->row_tiles = row_tiles_of(a, (size_t)forms[p->form].bt);
}

template <int TY, bool GATED>
static void mul_typed(const f8_mul_args *a, const f8_plan *p, hipStream_t s)
{
	/* a stream's workgroups take tile after tile */
	const size_t all = p->row_tiles * p->n_tiles, grid = p->form == TILE_256 && all > F8_CUS ? F8_CUS : all;
	const int n_tiles = (int)p->n_tiles, row_tiles = (int)p->row_tiles;
	switch (p->form) {
#define X(FORM, KERNEL, HALF, FP32, ...)                                                           \
	case FORM:                                                                                 \
		if constexpr (TY == HIP_F8_F32 ? FP32 : HALF)                                      \
			k_f8_##KERNEL<TY, GATED, __VA_ARGS__>                                      \
				<<<grid, p->threads, 0, s>>>(*a, n_tiles, row_tiles);              \
		break;
		F8_FORMS(X)
#undef X
	}
}

int f8_launch_mul(const f8_mul_args *a, const f8_plan *p, void *stream)
{
	hipStream_t s = (hipStream_t)stream;
	const bool gated = a->w[1] != NULL;
	if (p->type == HIP_F8_F32)
		gated ? mul_typed<HIP_F8_F32, true>(a, p, s) : mul_typed<HIP_F8_F32, false>(a, p, s);
	else if (p->type == HIP_F8_F16)
		gated ? mul_typed<HIP_F8_F16, true>(a, p, s) : mul_typed<HIP_F8_F16, false>(a, p, s);
	else
		gated ? mul_typed<HIP_F8_BF16, true>(a, p, s) : mul_typed<HIP_F8_BF16, false>(a, p, s);
	return hipGetLastError();
}
