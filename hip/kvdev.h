/*
 * nvshare-amd: device code that the paged key/value cache's kernels share.
 */
#ifndef NVS_KVDEV_H
#define NVS_KVDEV_H

#include <hip/hip_runtime.h>

#include <cstdint>

#include "kvcache.h"

typedef __bf16 bf16_t;
typedef _Float16 fp16_t;

struct e4m3_t {
	unsigned char bits;
};

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef bf16_t bf16x2 __attribute__((ext_vector_type(2)));
typedef fp16_t fp16x2 __attribute__((ext_vector_type(2)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef fp16_t fp16x8 __attribute__((ext_vector_type(8)));

template <typename T> struct types;
template <> struct types<bf16_t> {
	typedef bf16x2 x2;
	typedef bf16x8 x8;
	/* How far the running maximum of a softmax may lag behind, and what
	 * is added to each exponent, in powers of two (struct softmax). */
	static constexpr float lag = 8.f, lift = 0.f;
	static constexpr unsigned exponent = 0x7f807f80u, one = 0x00800080u;
};
template <> struct types<fp16_t> {
	typedef fp16x2 x2;
	typedef fp16x8 x8;
	/* Weights are at most 2^(11 + 4), below fp16's 2^16, and keep their
	 * 11 bits down to 2^-25 of the largest. */
	static constexpr float lag = 4.f, lift = 11.f;
	static constexpr unsigned exponent = 0x7c007c00u, one = 0x04000400u;
};

/* A number that is the same in the whole wave, where the compiler does not
 * see that it is. */
__device__ __forceinline__ int uniform(int x)
{
	return __builtin_amdgcn_readfirstlane(x);
}

__device__ __forceinline__ int64_t uniform64(int64_t x)
{
	return (int64_t)(((uint64_t)(unsigned)uniform((int)(x >> 32)) << 32) |
			 (unsigned)uniform((int)x));
}

/* Two numbers rounded to nearest, ties to even. */
template <typename T>
__device__ __forceinline__ unsigned pack2(float a, float b)
{
	typename types<T>::x2 v = { (T)a, (T)b };

	return __builtin_bit_cast(unsigned, v);
}

/* Two weights (0 or more), each as a number cut off after T's bits and the
 * rest of it, rounded to nearest: {both first parts, both rests}.  The rest
 * of a weight that is not 0 is not 0 either (what is added is at most 2^-20
 * of the weight, or T's smallest number), and no part is negative, so that
 * infinity times both is infinity. */
template <typename T>
__device__ __forceinline__ u32x2 split2(float a, float b)
{
	constexpr float MORE = 1.f + 0x1p-20f;

	if constexpr (__is_same(T, bf16_t)) {
		const unsigned u = __builtin_bit_cast(unsigned, a);
		const unsigned v = __builtin_bit_cast(unsigned, b);
		const float ha = __builtin_bit_cast(float, u & 0xffff0000u);
		const float hb = __builtin_bit_cast(float, v & 0xffff0000u);

		return u32x2{ u >> 16 | (v & 0xffff0000u),
			      pack2<T>(__builtin_fmaf(a, MORE, -ha),
				       __builtin_fmaf(b, MORE, -hb)) };
	} else {
		typedef unsigned short u16x2
			__attribute__((ext_vector_type(2)));
		const fp16x2 h = __builtin_bit_cast(
			fp16x2, __builtin_amdgcn_cvt_pkrtz(a, b));
		const u16x2 n = __builtin_bit_cast(u16x2, h);

		const unsigned rest =
			pack2<T>(__builtin_fmaf(a, MORE, -(float)h[0]),
				 __builtin_fmaf(b, MORE, -(float)h[1]));
		const u16x2 least = __builtin_elementwise_min(n, u16x2{ 1, 1 });

		return u32x2{ __builtin_bit_cast(unsigned, h),
			      rest | __builtin_bit_cast(unsigned, least) };
	}
}

/* Two e4m3 numbers as T: exact in both types. */
template <typename T, bool HIGH>
__device__ __forceinline__ unsigned widen2(unsigned w)
{
	if constexpr (__is_same(T, bf16_t))
		return __builtin_bit_cast(
			unsigned,
			__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f,
								  HIGH));
	else
		return __builtin_bit_cast(
			unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(
					  w, 1.f, HIGH));
}

template <typename T>
__device__ __forceinline__ u32x4 widen8(u32x2 w)
{
	return u32x4{ widen2<T, false>(w[0]), widen2<T, true>(w[0]),
		      widen2<T, false>(w[1]), widen2<T, true>(w[1]) };
}

/* The last b in [0, n] with f(b) <= x, for a rising f with f(0) <= x. */
template <typename F>
__device__ __forceinline__ int last_at_most(int n, int64_t x, F f)
{
	int lo = 0, hi = n;

	while (lo < hi) {
		int mid = lo + (hi - lo + 1) / 2;

		if (f(mid) <= x)
			lo = mid;
		else
			hi = mid - 1;
	}
	return lo;
}

/* A sequence's part of the step: rows first .. first + count - 1, the
 * first of them at position pos (which may be below zero). */
struct sequence {
	int first, count;
	int64_t pos;
};

__device__ __forceinline__ sequence sequence_of(const nvs_kv &c, int b)
{
	sequence s;

	if (c.starts) {
		s.first = c.starts[b];
		s.count = c.starts[b + 1] - s.first;
		/* Never beyond the rows, whatever starts holds: a sequence
		 * that would be has none of them. */
		if (s.first < 0 || s.count < 0 || s.first > c.total ||
		    s.count > c.total - s.first)
			s.count = 0;
	} else {
		s.count = c.total / c.batch;
		s.first = b * s.count;
	}
	s.pos = (int64_t)c.lens[b] - s.count;
	return s;
}

/* The sequence of a row; -1 where it belongs to none. */
__device__ __forceinline__ int sequence_at(const nvs_kv &c, int row)
{
	if (!c.starts)
		return row / (c.total / c.batch);
	const int *starts = c.starts;

	if (starts[0] > row)
		return -1;
	const int b = last_at_most(c.batch, row,
				   [=](int i) { return (int64_t)starts[i]; });
	return b == c.batch ? -1 : b;
}

#endif
