/*
 * nvshare-amd gfx950 kernels of a paged key/value cache
 * (libnvshare_hiputil.so): what an interactive session holds on the GPU
 * between two bursts, and so what the interposer pages out and back.
 *
 *   nvs_kv_append   stores new keys and values in the cache's pages and
 *                   rotates new queries and keys by their positions
 *   nvs_kv_attend   attention of a step's new tokens over the cache
 *
 * Sequence b holds lens[b] tokens, its newest n_b are the call's rows
 * starts[b] .. starts[b + 1] - 1 (without starts: total / batch rows
 * each).  Row i of them has position p = lens[b] - n_b + i; position j
 * lies in slot j % page_size of page table[b][j / page_size].
 *
 * lens, starts and the table are read on the device, so a captured graph
 * follows them; every index made from them is checked there.  An entry
 * outside [0, pages) is no page: nothing is stored in it and nothing of
 * it is attended to.
 */
#include <hip/hip_runtime.h>

#include <cstdint>

#include "kvcache.h"

namespace {

typedef __bf16 bf16_t;
typedef _Float16 fp16_t;
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

struct e4m3_t {
	unsigned char bits;
};

template <typename T> struct vec8 {
	T x[8];
};

__device__ __forceinline__ float to_f32(bf16_t x)
{
	return (float)x;
}

__device__ __forceinline__ float to_f32(fp16_t x)
{
	return (float)x;
}

__device__ __forceinline__ float to_f32(e4m3_t x)
{
	return __builtin_amdgcn_cvt_f32_fp8((int)x.bits, 0);
}

/* Eight values from 16 aligned bytes (8 of e4m3). */
template <typename T>
__device__ __forceinline__ void load8(const T *p, float *x)
{
	if constexpr (sizeof(T) == 1) {
		u32x2 w = *(const u32x2 *)p;
#pragma unroll
		for (int i = 0; i < 2; i++) {
			f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(w[i], false);
			f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(w[i], true);
			x[4 * i] = lo[0];
			x[4 * i + 1] = lo[1];
			x[4 * i + 2] = hi[0];
			x[4 * i + 3] = hi[1];
		}
	} else {
		vec8<T> v = __builtin_bit_cast(vec8<T>, *(const u32x4 *)p);
#pragma unroll
		for (int i = 0; i < 8; i++)
			x[i] = (float)v.x[i];
	}
}

/* Rounded to nearest, ties to even: the one rounding of each result. */
template <typename T>
__device__ __forceinline__ void store8(T *p, const float *x)
{
	vec8<T> v;
#pragma unroll
	for (int i = 0; i < 8; i++)
		v.x[i] = (T)x[i];
	*(u32x4 *)p = __builtin_bit_cast(u32x4, v);
}

/* e4m3 has no infinity: what is over its largest value, 448, is held as
 * that; a NaN stays one. */
__device__ __forceinline__ float e4m3_range(float x)
{
	return x != x ? x : fminf(fmaxf(x, -448.f), 448.f);
}

__device__ __forceinline__ void store8(e4m3_t *p, const float *x)
{
	u32x2 w;
#pragma unroll
	for (int i = 0; i < 2; i++) {
		int r = 0;

		r = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_range(x[4 * i]),
						    e4m3_range(x[4 * i + 1]),
						    r, false);
		r = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_range(x[4 * i + 2]),
						    e4m3_range(x[4 * i + 3]),
						    r, true);
		w[i] = r;
	}
	*(u32x2 *)p = w;
}

/* The place of a row: its sequence and position.  seq is -1 for a row
 * that belongs to no sequence (padding behind the last one). */
struct place {
	int seq;
	int64_t pos;
};

__device__ __forceinline__ place place_of(const nvs_kv &c, int row)
{
	int first, count, b;

	if (c.starts) {
		/* The last b with starts[b] <= row. */
		int lo = 0, hi = c.batch; /* in [lo, hi] */

		while (lo < hi) {
			int mid = (lo + hi + 1) >> 1;

			if (c.starts[mid] <= row)
				lo = mid;
			else
				hi = mid - 1;
		}
		if (lo == c.batch || c.starts[lo] > row)
			return { -1, 0 };
		b = lo;
		first = c.starts[b];
		count = c.starts[b + 1] - first;
	} else {
		count = c.total / c.batch;
		b = row / count;
		first = b * count;
	}
	return { b, (int64_t)c.lens[b] - count + (row - first) };
}

/* ------------------------------------------------------------------ */
/* append                                                              */
/* ------------------------------------------------------------------ */

/*
 * (x1, x2) -> (x1 cos - x2 sin, x2 cos + x1 sin) for each pair of the
 * first `rotary` dimensions of queries and keys, in 32 bits; values are
 * moved as they are.
 *
 * A thread takes 16 dimensions of one head: two pieces of 8, the halves
 * of 8 pairs, so that every access is 16 bytes and a thread needs 8
 * cosines and sines only.
 */
template <typename T, typename C>
__global__ __launch_bounds__(256) void append_kernel(nvs_kv c,
						     nvs_kv_append_args a)
{
	const int units = c.dim / 16;
	const int q_heads = a.q ? c.heads : 0;
	const int all = q_heads + 2 * c.kv_heads;
	int64_t w = (int64_t)blockIdx.x * 256 + threadIdx.x;
	const int u = w % units;
	w /= units;
	const int head = w % all;
	const int64_t row64 = w / all;

	if (row64 >= c.total)
		return;
	const int row = (int)row64;
	const place at = place_of(c, row);
	const int64_t capacity = (int64_t)c.per_seq * c.page_size;
	const bool in_range = at.seq >= 0 && at.pos >= 0 && at.pos < capacity;
	const int kind = head < q_heads ? 0 :
			 head < q_heads + c.kv_heads ? 1 : 2;
	const int h = kind == 0 ? head : kind == 1 ? head - q_heads :
		      head - q_heads - c.kv_heads;
	const bool turn = kind < 2 && a.rotation && 16 * u < a.rotary;
	int e0 = 16 * u, e1 = 16 * u + 8;

	if (turn && !a.interleaved) {
		e0 = 8 * u;
		e1 = 8 * u + a.rotary / 2;
	}

	if (!in_range) {
		/* No token: queries give zeros in a buffer of our own. */
		if (kind == 0 && (at.seq >= 0 || a.fill)) {
			float zero[8] = {};
			T *o = (T *)a.q_out + row * a.q_out_row +
			       h * a.q_out_head;

			store8(o + e0, zero);
			store8(o + e1, zero);
		}
		return;
	}

	const T *src = kind == 0 ?
			       (const T *)a.q + row * a.q_row + h * a.q_head :
		       kind == 1 ?
			       (const T *)a.k + row * a.k_row + h * a.k_head :
			       (const T *)a.v + row * a.v_row + h * a.v_head;
	float x0[8], x1[8];

	load8(src + e0, x0);
	load8(src + e1, x1);
	if (turn) {
		const float *cs = a.rotation + at.pos * a.rotation_row + 8 * u;
		const float *sn = cs + a.rotary / 2;

		if (a.interleaved) {
#pragma unroll
			for (int i = 0; i < 8; i++) {
				float *p = i < 4 ? x0 + 2 * i : x1 + 2 * i - 8;
				float p0 = p[0], p1 = p[1];

				p[0] = p0 * cs[i] - p1 * sn[i];
				p[1] = p1 * cs[i] + p0 * sn[i];
			}
		} else {
#pragma unroll
			for (int i = 0; i < 8; i++) {
				float p0 = x0[i], p1 = x1[i];

				x0[i] = p0 * cs[i] - p1 * sn[i];
				x1[i] = p1 * cs[i] + p0 * sn[i];
			}
		}
	}
	if (kind == 0) {
		T *o = (T *)a.q_out + row * a.q_out_row + h * a.q_out_head;

		store8(o + e0, x0);
		store8(o + e1, x1);
		return;
	}

	const int entry = (int)(at.pos / c.page_size);
	const int slot = (int)(at.pos % c.page_size);
	const int page = c.table[at.seq * c.table_row + entry];

	if ((unsigned)page >= (unsigned)c.pages)
		return;
	const int64_t off = kind == 1 ?
				    page * c.k_page + slot * c.k_slot +
					    h * c.k_head :
				    page * c.v_page + slot * c.v_slot +
					    h * c.v_head;
	C *dst = (C *)(kind == 1 ? c.k_cache : c.v_cache) + off;

	if constexpr (sizeof(C) == 1) {
		const float s = kind == 1 ? c.k_scale[h] : c.v_scale[h];
#pragma unroll
		for (int i = 0; i < 8; i++) {
			x0[i] /= s;
			x1[i] /= s;
		}
	}
	store8(dst + e0, x0);
	store8(dst + e1, x1);
}

/* ------------------------------------------------------------------ */
/* attend                                                              */
/* ------------------------------------------------------------------ */

/*
 * One wave to a query row and head, 64 keys at a time with the running
 * maximum and sum of the softmax in 32 bits: a lane has a key while the
 * scores are made, and dimensions while the values are added.
 */
template <typename T, typename C>
__global__ __launch_bounds__(64) void attend_kernel(nvs_kv c, nvs_kv_attend_args a)
{
	__shared__ float q[256], p[64];
	__shared__ int64_t where[64];
	const int row = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
	const int kh = h / (c.heads / c.kv_heads);
	const place at = place_of(c, row);
	T *out = (T *)a.out + row * a.out_row + h * a.out_head;

	if (at.seq < 0) {
		if (a.fill)
			for (int d = lane; d < c.dim; d += 64)
				out[d] = (T)0.f;
		if (a.lse && lane == 0)
			a.lse[(int64_t)row * c.heads + h] = -INFINITY;
		return;
	}
	const int64_t capacity = (int64_t)c.per_seq * c.page_size;
	const int64_t end = min(at.pos + 1, capacity);
	const int64_t begin = a.window > 0 && at.pos + 1 > a.window ?
				      at.pos + 1 - a.window : 0;
	const T *src = (const T *)a.q + row * a.q_row + h * a.q_head;
	const float ks = c.k_scale ? c.k_scale[kh] : 1.f;
	const float vs = c.v_scale ? c.v_scale[kh] : 1.f;
	float top = -INFINITY, sum = 0.f, acc[4] = {};

	for (int d = lane; d < c.dim; d += 64)
		q[d] = to_f32(src[d]) * a.scale * ks;
	__syncthreads();
	for (int64_t j0 = begin; j0 < end; j0 += 64) {
		const int64_t j = j0 + lane;
		float s = -INFINITY;
		int page = -1;

		if (j < end)
			page = c.table[at.seq * c.table_row + j / c.page_size];
		const bool seen = (unsigned)page < (unsigned)c.pages;
		const int64_t slot = j % c.page_size;

		where[lane] = -1;
		if (seen) {
			const C *k = (const C *)c.k_cache + page * c.k_page +
				     slot * c.k_slot + kh * c.k_head;

			s = 0.f;
			for (int d = 0; d < c.dim; d += 8) {
				float x[8];

				load8(k + d, x);
				for (int i = 0; i < 8; i++)
					s += q[d + i] * x[i];
			}
			where[lane] = page * c.v_page + slot * c.v_slot +
				      kh * c.v_head;
		}
		float m = s;
		for (int o = 32; o; o >>= 1)
			m = fmaxf(m, __shfl_xor(m, o));
		m = fmaxf(m, top);
		const float base = m == -INFINITY ? 0.f : m;
		const float e = seen ? expf(s - base) : 0.f;
		const float keep = expf(top - base);
		float t = e;
		for (int o = 32; o; o >>= 1)
			t += __shfl_xor(t, o);
		sum = sum * keep + t;
		top = m;
		p[lane] = e;
		__syncthreads();
		for (int i = 0; i < 4; i++)
			acc[i] *= keep;
		for (int n = 0; n < 64; n++) {
			if (where[n] < 0)
				continue;
			const C *v = (const C *)c.v_cache + where[n];

			for (int i = 0; i < 4; i++)
				if (lane + 64 * i < c.dim)
					acc[i] += p[n] *
						  to_f32(v[lane + 64 * i]);
		}
		__syncthreads();
	}
	for (int i = 0; i < 4; i++)
		if (lane + 64 * i < c.dim)
			out[lane + 64 * i] =
				(T)(sum == 0.f ? 0.f : acc[i] / sum * vs);
	if (a.lse && lane == 0)
		a.lse[(int64_t)row * c.heads + h] =
			sum == 0.f ? -INFINITY : top + logf(sum);
}

bool aligned(const void *p, int64_t bytes)
{
	return ((uintptr_t)p & (bytes - 1)) == 0;
}

/* What every access of the kernels relies on. */
bool sound(const nvs_kv &c)
{
	const int size = c.cache_type == NVS_KV_E4M3 ? 1 : 2;
	const int64_t strides = c.k_page | c.k_slot | c.k_head | c.v_page |
				c.v_slot | c.v_head;

	return c.batch > 0 && c.total >= 0 && c.heads > 0 && c.kv_heads > 0 &&
	       c.heads % c.kv_heads == 0 && c.pages > 0 && c.page_size > 0 &&
	       c.per_seq > 0 && c.k_cache && c.v_cache && c.lens && c.table &&
	       (c.type == NVS_KV_BF16 || c.type == NVS_KV_FP16) &&
	       (c.cache_type == c.type || c.cache_type == NVS_KV_E4M3) &&
	       (size == 2 || (c.k_scale && c.v_scale)) &&
	       (c.starts || c.total % c.batch == 0) &&
	       (strides * size) % 16 == 0 && aligned(c.k_cache, 16) &&
	       aligned(c.v_cache, 16);
}

template <typename T, typename C>
int launch_append(const nvs_kv &c, const nvs_kv_append_args &a, hipStream_t s)
{
	const int64_t all = (a.q ? c.heads : 0) + 2 * c.kv_heads;
	const int64_t n = c.total * all * (c.dim / 16);

	hipLaunchKernelGGL((append_kernel<T, C>), dim3((n + 255) / 256),
			   dim3(256), 0, s, c, a);
	return (int)hipGetLastError();
}

template <typename T, typename C>
int launch_attend(const nvs_kv &c, const nvs_kv_attend_args &a, hipStream_t s)
{
	hipLaunchKernelGGL((attend_kernel<T, C>), dim3(c.total, c.heads),
			   dim3(64), 0, s, c, a);
	return (int)hipGetLastError();
}

} /* namespace */

/* F(T, C, ...) for the types of the queries and of the cache. */
#define BY_TYPE(F, c, ...)                                                 \
	((c).type == NVS_KV_BF16 ?                                         \
		 ((c).cache_type == NVS_KV_E4M3 ?                          \
			  F<bf16_t, e4m3_t>(c, __VA_ARGS__) :              \
			  F<bf16_t, bf16_t>(c, __VA_ARGS__)) :             \
		 ((c).cache_type == NVS_KV_E4M3 ?                          \
			  F<fp16_t, e4m3_t>(c, __VA_ARGS__) :              \
			  F<fp16_t, fp16_t>(c, __VA_ARGS__)))

extern "C" {

int nvs_kv_append(const nvs_kv *c, const nvs_kv_append_args *a, void *stream)
{
	if (!c || !a || !sound(*c) || c->dim <= 0 || c->dim % 16 ||
	    !a->k || !a->v || (a->q && !a->q_out) ||
	    (a->rotation && (a->rotary <= 0 || a->rotary % 16 ||
			     a->rotary > c->dim)))
		return (int)hipErrorInvalidValue;
	if ((a->q_row | a->q_head | a->k_row | a->k_head | a->v_row |
	     a->v_head | a->q_out_row | a->q_out_head) % 8 ||
	    !aligned(a->q, 16) || !aligned(a->k, 16) || !aligned(a->v, 16) ||
	    !aligned(a->q_out, 16) || !aligned(a->rotation, 16) ||
	    a->rotation_row % 4)
		return (int)hipErrorInvalidValue;
	if (c->total == 0)
		return 0;
	return BY_TYPE(launch_append, *c, *a, (hipStream_t)stream);
}

int nvs_kv_attend(const nvs_kv *c, const nvs_kv_attend_args *a, void *stream)
{
	if (!c || !a || !sound(*c) ||
	    (c->dim != 64 && c->dim != 128 && c->dim != 256) || !a->q ||
	    !a->out || a->window < 0)
		return (int)hipErrorInvalidValue;
	if ((a->q_row | a->q_head | a->out_row | a->out_head) % 8 ||
	    !aligned(a->q, 16) || !aligned(a->out, 16))
		return (int)hipErrorInvalidValue;
	if (c->total == 0)
		return 0;
	return BY_TYPE(launch_attend, *c, *a, (hipStream_t)stream);
}

} /* extern "C" */
