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
#include "kvdev.h"
#include "kvattend.h"

namespace {

template <typename T> struct vec8 {
	T x[8];
};

/* Eight values from 16 aligned bytes. */
template <typename T>
__device__ __forceinline__ void load8(const T *p, float *x)
{
	const vec8<T> v = __builtin_bit_cast(vec8<T>, *(const u32x4 *)p);

#pragma unroll
	for (int i = 0; i < 8; i++)
		x[i] = (float)v.x[i];
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

/* ------------------------------------------------------------------ */
/* append                                                              */
/* ------------------------------------------------------------------ */

/*
 * (x1, x2) -> (x1 cos - x2 sin, x2 cos + x1 sin) for each pair of the
 * first `rotary` dimensions of queries and keys, in 32 bits; values are
 * moved as they are.
 *
 * Bound by bytes, each read and written once.  A thread takes 16
 * dimensions of one head: two pieces of 8, the halves of 8 pairs, so that
 * every access is 16 bytes and a thread needs 8 cosines and sines only;
 * these are shared by a row's heads and come from cache.  15512 rows (32
 * query heads, 8 cached ones of 128, 389 MB): 85 us, 4.56 TB/s, as fast as
 * a copy of 4 GiB; one row: 3.0 us, a call 5.7.
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
	int b = sequence_at(c, row);
	int64_t pos = -1;

	if (b >= 0) {
		const sequence s = sequence_of(c, b);

		if (row - s.first < s.count)
			pos = s.pos + (row - s.first);
		else
			b = -1;
	}
	const int capacity = c.per_seq * c.page_size;
	const bool in_range = pos >= 0 && pos < capacity;
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
		if (kind == 0 && (b >= 0 || a.fill)) {
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
		const float *cs = a.rotation + pos * a.rotation_row + 8 * u;
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

	const int entry = (int)(pos / c.page_size);
	const int slot = (int)(pos % c.page_size);
	const int page = c.table[b * c.table_row + entry];

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
	       (int64_t)c.total * c.heads < 0x7fffffff &&
	       (int64_t)c.per_seq * c.page_size <= 0x7fffffff &&
	       c.per_seq > 0 && c.k_cache && c.v_cache && c.lens && c.table &&
	       (c.type == NVS_KV_BF16 || c.type == NVS_KV_FP16) &&
	       (c.cache_type == c.type || c.cache_type == NVS_KV_E4M3) &&
	       (size == 2 || (c.k_scale && c.v_scale)) &&
	       (c.starts || c.total % c.batch == 0) &&
	       (strides * size) % 16 == 0 && aligned(c.k_cache, 16) &&
	       aligned(c.v_cache, 16);
}

/* A grid's threads are counted in 32 bits. */
bool too_large(int64_t blocks, int64_t threads)
{
	return blocks * threads > 0xffffffffll;
}

template <typename T, typename C>
int launch_append(const nvs_kv &c, const nvs_kv_append_args &a, hipStream_t s)
{
	const int64_t all = (a.q ? c.heads : 0) + 2 * c.kv_heads;
	const int64_t n = c.total * all * (c.dim / 16);

	if (too_large((n + 255) / 256, 256))
		return (int)hipErrorInvalidValue;
	hipLaunchKernelGGL((append_kernel<T, C>), dim3((n + 255) / 256),
			   dim3(256), 0, s, c, a);
	return (int)hipGetLastError();
}

bool sound_attend(const nvs_kv &c, const nvs_kv_attend_args &a)
{
	return (c.dim == 64 || c.dim == 128 || c.dim == 256) && a.q && a.out &&
	       a.window >= 0 && a.max_new >= 0 &&
	       (a.q_row | a.q_head | a.out_row | a.out_head) % 8 == 0 &&
	       aligned(a.q, 16) && aligned(a.out, 16);
}

int64_t ceil_div(int64_t a, int64_t b)
{
	return (a + b - 1) / b;
}

/*
 * The division of a call's work, by what the host knows: rows, sequences,
 * the table's width and the most rows that a sequence may have.  With few
 * blocks of rows, the keys are divided so that there are enough blocks for
 * 256 CUs to be evenly loaded.
 */
nvs_plan plan_of(const nvs_kv &c, const nvs_kv_attend_args &a, void *work,
		 int64_t &bytes)
{
	const int64_t group = c.heads / c.kv_heads;
	const int64_t most_new = c.starts ? a.max_new : c.total / c.batch;
	const int64_t most_rows = most_new * group;
	int64_t keys = (int64_t)c.per_seq * c.page_size;
	nvs_plan p = {};

	if (a.window > 0)
		keys = keys < a.window + most_new ? keys : a.window + most_new;
	/* With 2^(l - 1) < page_size <= 2^l, ceil(2^(31 + l) / page_size)
	 * divides numbers of 31 bits. */
	int l = 0;

	while (1ll << l < c.page_size)
		l++;
	p.page_shift = 31 + l;
	p.page_magic = ((1ull << p.page_shift) + c.page_size - 1) /
		       (uint64_t)c.page_size;
	const int64_t slot = c.k_slot > c.v_slot ? c.k_slot : c.v_slot;

	p.near_slots = slot < (1ll << 30) / WIDE_TILE;
	/* Two columns of 16 rows are what a narrow block holds.  For 32 rows
	 * of each sequence, narrow and wide take: 8 sequences over 5000 keys,
	 * heads of 128, 45 and 46 us, e4m3 33 and 46; one over 5000, 22 and
	 * 35; 16 over 16000, 199 and 190; 8 over 5000 with heads of 256, 129
	 * and 98 (registers spill in the narrow kernel), e4m3 88 and 95.  20
	 * rows: 44 and 45.
	 *
	 * Among longer sequences one column only, as single tokens have.
	 * Two: prompts and single tokens 398 us instead of 395; but 24
	 * sequences of 4 to 32 rows over up to 5000 keys, in a step that may
	 * have longer ones, 79 instead of 109, over up to 30000 246 instead of
	 * 462. */
	p.span = most_rows > 32 || most_rows <= 16 ? 16 : 32;
	p.narrow_rows = most_rows <= 32 ? 0x7fffffff : c.starts ? 16 : 0;
	p.joined_rows = (int)(most_rows < p.span ? most_rows : p.span);
	p.narrow_blocks = p.narrow_rows ? 1 : 0;
	p.wide_parts = 1;
	if (p.narrow_rows && p.joined_rows) {
		/* As many blocks as the card holds at a time (2 a CU, 4 of
		 * the smallest rows): all begin and end together.  Twice as
		 * many take 390 us where these take 383, for 64 tokens over
		 * 8192 keys each, and 39 where these take 33, over 500. */
		const int size = c.cache_type == NVS_KV_E4M3 ? 1 : 2;
		const int64_t tile = nvs_narrow_tile(c.dim, size);
		const int64_t most = ceil_div(
			c.batch * ceil_div(keys, tile), NARROW_LEAST);
		const int64_t want = (c.dim * size < 128 ? 1024 : 512) /
				     c.kv_heads;

		p.narrow_blocks = (int)(most < want ? most :
					want > 1   ? want :
						     1);
		/* Short sequences go to a block each, and no join is wanted:
		 * with two tiles to a wave always (one token over 200 keys:
		 * 9.2 us, 12.1 divided), with four where there are enough to
		 * fill the card (64 over 500: 28.8, 32.5 divided; one: 13.7,
		 * 10.9 divided). */
		const int64_t turns =
			ceil_div(ceil_div(keys, tile),
				 nvs_narrow_waves(c.dim, size));

		if (turns <= 2 ||
		    (turns <= 4 && (int64_t)c.batch * c.kv_heads >= 256)) {
			p.narrow_blocks = c.batch;
			p.narrow_whole = 1;
		}
	}
	if (most_rows > 32) {
		p.wide_blocks =
			(int)(c.starts ? c.total * group / WIDE_ROWS + c.batch :
					 c.batch *
						 ceil_div(most_rows, WIDE_ROWS));
		/* Two blocks a CU.  A block of rows sees no more keys than
		 * its window and its own tokens. */
		const int64_t want =
			512 / ((int64_t)p.wide_blocks * c.kv_heads);
		const int64_t seen = a.window + WIDE_ROWS / group + 1;
		const int64_t most =
			ceil_div(a.window > 0 && seen < keys ? seen : keys,
				 WIDE_TILE) /
			WIDE_LEAST;

		p.wide_parts = (int)(want < most ? want : most);
		if (p.wide_parts < 1)
			p.wide_parts = 1;
	}
	/* The parts' results, narrow before wide. */
	const int64_t narrow = p.narrow_blocks > 1 && !p.narrow_whole ?
				       (int64_t)p.narrow_blocks * 2 *
					       c.kv_heads * p.span :
				       0;
	const int64_t wide = p.wide_parts > 1 ? (int64_t)p.wide_parts *
							c.total * c.heads :
						0;

	p.narrow_out = (float *)work;
	p.wide_out = p.narrow_out + narrow * c.dim;
	p.narrow_sum = (f32x2 *)(p.wide_out + wide * c.dim);
	p.wide_sum = p.narrow_sum + narrow;
	bytes = (narrow + wide) * (c.dim * 4 + 8);
	if (narrow) {
		p.tiles_at = (int64_t *)(p.wide_sum + wide);
		bytes += (c.batch + 1ll) * 8;
	}
	return p;
}

template <typename T, typename C>
int launch_attend(const nvs_kv &c, const nvs_kv_attend_args &a,
		  const nvs_plan &p, hipStream_t s)
{
	hipError_t e = hipSuccess;

	if (p.narrow_rows)
		e = nvs_narrow<T, C>(c, a, p, s);
	if (e == hipSuccess && p.wide_blocks)
		e = nvs_wide<T, C>(c, a, p, s);
	if (e == hipSuccess && p.narrow_blocks > 1 && !p.narrow_whole)
		e = nvs_join<T>(c, a, p, true, s);
	if (e == hipSuccess && p.wide_parts > 1)
		e = nvs_join<T>(c, a, p, false, s);
	return (int)e;
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

/* Bytes that nvs_kv_attend needs at `work`; -1: refused. */
int64_t nvs_kv_attend_work(const nvs_kv *c, const nvs_kv_attend_args *a)
{
	int64_t bytes;

	if (!c || !a || !sound(*c) || !sound_attend(*c, *a))
		return -1;
	if (c->total == 0)
		return 0;
	plan_of(*c, *a, nullptr, bytes);
	return bytes;
}

int nvs_kv_attend(const nvs_kv *c, const nvs_kv_attend_args *a, void *work,
		  void *stream)
{
	int64_t bytes;

	if (!c || !a || !sound(*c) || !sound_attend(*c, *a))
		return (int)hipErrorInvalidValue;
	if (c->total == 0)
		return 0;
	const nvs_plan p = plan_of(*c, *a, work, bytes);

	if ((bytes && (!work || !aligned(work, 16))) ||
	    too_large((int64_t)p.narrow_blocks * c->kv_heads, 256) ||
	    too_large((int64_t)p.wide_blocks * c->kv_heads * p.wide_parts,
		      256) ||
	    too_large((int64_t)c->batch * c->kv_heads * p.joined_rows, 64) ||
	    (p.wide_parts > 1 && too_large((int64_t)c->total * c->heads, 64)))
		return (int)hipErrorInvalidValue;
	return BY_TYPE(launch_attend, *c, *a, p, (hipStream_t)stream);
}

} /* extern "C" */
