/*
 * Device helpers of the rotary positions and the 4-bit cache: the values of
 * the three activation types, and where a row of a sequence lies in the pool.
 * The layout of a tile is include/hip_kv.h's.
 */
#ifndef KV_DEVICE_H
#define KV_DEVICE_H

#include "moe_device.h"
#include "kv_internal.h"

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx8 __attribute__((ext_vector_type(8)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef unsigned short ushort2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <int TY> struct kv_type;
template <> struct kv_type<HIP_KV_F32> {
	typedef float t;
	__device__ static float get(t v) { return v; }
	__device__ static t put(float v) { return v; }
};
template <> struct kv_type<HIP_KV_F16> {
	typedef _Float16 t;
	__device__ static float get(t v) { return (float)v; }
	__device__ static t put(float v) { return (_Float16)v; }
};
template <> struct kv_type<HIP_KV_BF16> {
	typedef __bf16 t;
	__device__ static float get(t v) { return (float)v; }
	__device__ static t put(float v) { return (__bf16)v; }
};

/* N consecutive values of a type, as one aligned load or store where they
 * are 8 or 16 bytes */
template <int TY, int N> struct __attribute__((aligned(sizeof(typename kv_type<TY>::t) * N >= 16
				? 16 : sizeof(typename kv_type<TY>::t) * N))) kv_vec {
	typename kv_type<TY>::t v[N];
};

/* sizes and offsets inside a tile of 32 rows of heads of D channels */
template <int D> struct kv_tile {
	static constexpr int G = D / 32;          /* key groups of a row */
	static constexpr int P = G < 4 ? G : 4;   /* words of a lane that follow each other */
	static constexpr int V_CODES = 16 * D;    /* byte offsets */
	static constexpr int K_SCALES = 32 * D;
	static constexpr int V_SCALES = 34 * D;
	static constexpr int BYTES = 34 * D + 64;
	/* word of key codes: row r, channel c (its 8 channels c / 8 * 8 ..) */
	__device__ static int k_word(int r, int c)
	{
		const int g = c / 32, part = c % 32 / 8;
		return ((r / 16 * (G / P) + g / P) * 64 + part * 16 + r % 16) * P + g % P;
	}
	/* word of value codes, from V_CODES on: channel c, row r (its 8 rows) */
	__device__ static int v_word(int r, int c)
	{
		return (c / 64 * 64 + r % 16 / 4 * 16 + c % 16) * 4 + c / 16 % 4;
	}
	/* which of a value word's 8 codes row r is */
	__device__ static int v_code(int r) { return r % 4 + r / 16 * 4; }
};

/* where code j of a word starts; the word turned right by that has it in its
 * low four bits */
__device__ static inline int kv_bit(int j)
{
	return 2 + 4 * (j >> 1) + 16 * (j & 1);
}

__device__ static inline u32 kv_rotr(u32 v, int n)
{
	return __builtin_amdgcn_alignbit(v, v, n);
}

/* a sequence of the batch: its first row, rows and length, cut to the
 * batch's bounds */
struct kv_seq {
	int row, n, len;
};

__device__ static inline void kv_error(const kv_args &a, u32 bit)
{
	if (a.err)
		atomicOr(a.err, bit);
}

__device__ static inline kv_seq kv_sequence(const kv_args &a, int s, bool report)
{
	kv_seq q;
	int end;
	if (a.row_start) {
		q.row = a.row_start[s];
		end = a.row_start[s + 1];
	} else {
		q.row = s * a.max_rows; /* at most rows, which the host checks */
		end = q.row + a.max_rows;
	}
	q.len = a.len[s];
	bool bad = false;
	if (q.row < 0 || q.row > a.rows || end < q.row || end > a.rows || end - q.row > a.max_rows) {
		bad = true;
		q.row = min(max(q.row, 0), a.rows);
		end = min(max(end, q.row), a.rows);
		end = min(end, q.row + a.max_rows);
	}
	if (q.len < 0 || q.len > a.max_len) {
		bad = true;
		q.len = min(max(q.len, 0), a.max_len);
	}
	if (bad && report)
		kv_error(a, HIP_KV_ERR_BATCH);
	q.n = end - q.row;
	return q;
}

__device__ static inline kv_seq kv_sequence(const kv_args &a, int s)
{
	return kv_sequence(a, s, threadIdx.x == 0);
}

/* tile t (rows 32 t ..) of kv head h of sequence s, NULL where its page is
 * not in the pool; t is below max_len / 32, rounded up */
template <int D>
__device__ static inline uint8_t *kv_tile_at(const kv_args &a, int s, int h, int t)
{
	const int shift = a.page_shift - 5; /* log2 of a page's tiles */
	const int id = a.table[s * a.table_stride + (t >> shift)];
	if ((u32)id >= (u32)a.pages)
		return NULL;
	const size_t tile = (((size_t)id * a.kv_heads + h) << shift) + (t & ((1 << shift) - 1));
	return a.pool + tile * kv_tile<D>::BYTES;
}

/* whether a launch has as many workgroups along x: below 2^32 threads */
static inline bool kv_launchable(size_t workgroups, int threads)
{
	return workgroups <= 0xffffffffu / (unsigned)threads;
}

#define KV_DISPATCH_TYPE(ty, TY, ...)                                             \
	switch (ty) {                                                             \
	case HIP_KV_F32: { constexpr int TY = HIP_KV_F32; __VA_ARGS__; break; }   \
	case HIP_KV_F16: { constexpr int TY = HIP_KV_F16; __VA_ARGS__; break; }   \
	default: { constexpr int TY = HIP_KV_BF16; __VA_ARGS__; break; }          \
	}

#define KV_DISPATCH_HEAD(d, D, ...)                                               \
	switch (d) {                                                              \
	case 64: { constexpr int D = 64; __VA_ARGS__; break; }                    \
	case 128: { constexpr int D = 128; __VA_ARGS__; break; }                  \
	default: { constexpr int D = 256; __VA_ARGS__; break; }                   \
	}

#endif
