/*
 * nvshare-amd: what the attention kernels share.
 *
 * Rows and work.  The query heads of one cached head are rows of the same
 * product: a sequence with n new tokens and G = heads / kv_heads has n * G
 * rows for each cached head, row r being token r / G and head r % G.  Two
 * kernels take blocks of these rows:
 *
 *   narrow  up to 32 rows, as single tokens and drafts have: its waves
 *           share the rows and divide the keys, so that the cache streams
 *           through all of them; bound by the cache's bytes.  Weights meet
 *           the values in two parts of the rows' type
 *   wide    128 rows, as chunks have: its waves divide the rows and share
 *           the keys in LDS; bound by the matrix products.  Weights are
 *           rounded once to the rows' type
 *
 * Both walk the keys in tiles with the running maximum and sum of the
 * softmax in 32 bits, and where there are few blocks of rows the keys are
 * divided between `parts` blocks, whose results a third kernel joins in
 * the order of the keys: no atomics, the same bits each time.
 *
 * Both compute S^T = K Q^T and O^T = V^T P^T, so that a lane has scores of
 * one row only: maxima and sums need no more than an exchange between the
 * wave's halves or quarters, and P^T is already laid out as the second
 * product's operand.  V^T comes from LDS by transposing reads.
 */
#ifndef NVS_KVATTEND_H
#define NVS_KVATTEND_H

#include "kvdev.h"

constexpr int WIDE_TILE = 64, WIDE_ROWS = 128;

constexpr int nvs_narrow_tile(int dim, int size)
{
	return dim * size < 256 ? 64 : 32;
}

/*
 * The fewest tiles that are worth a block of their own.
 *
 * Narrow: one for each of its waves.  With 2, one token over 611 keys takes
 * 11.9 us instead of 11.6 and 8 of 900 keys 15.3 instead of 19.8, with 8
 * 15.7 and 19.8; drafts of 6 over 5009 keys 21.2, 21.2 and 27.5.
 *
 * Wide: a join costs 4 to 5 us and the parts' traffic, and a block of heads
 * of 256 fills a CU, so that twice as many blocks take two rounds: two
 * chunks of 1500 in a window of 1024, 75 us with 16 or 32 and 106 with 4 or
 * 8.  With heads of 128 fewer are better where there are few blocks: one
 * sequence's 64 rows over 4000 keys 28, 25, 40 and 96 us with 4, 8, 16 and
 * 32; 800 rows over 2000 keys 29, 28, 39 and 55; 2048 over 4000 59, 59, 64
 * and 107; 8 sequences of 40 rows over 4000 36, 36, 42 and 95; long chunks
 * do not care.
 */
constexpr int NARROW_LEAST = 4, WIDE_LEAST = 16;
constexpr int nvs_narrow_waves(int dim, int size)
{
	return dim * size > 256 ? 2 : 4;
}

/* How the work of one call is divided. */
struct nvs_plan {
	int narrow_rows; /* sequences with more rows go to the wide kernel */
	int span;	 /* rows of a narrow block, 16 or 32 */
	int joined_rows; /* rows of a sequence that may be divided there */
	int narrow_blocks; /* narrow blocks for one cached head */
	int narrow_whole;  /* each of them has one sequence, undivided */
	int wide_blocks;   /* blocks of rows, for one cached head */
	int wide_parts;	   /* wide blocks that may divide one's keys */
	uint64_t page_magic; /* key / page_size = key * magic >> shift */
	int page_shift;
	int near_slots; /* a tile's rows lie within 31 bits of each other */
	/* Results and (log2 of the weights' unit, sum of the weights in it)
	 * of parts: of narrow blocks by part_at(), of wide ones by [part]
	 * [row][head]. */
	float *narrow_out, *wide_out;
	f32x2 *narrow_sum, *wide_sum;
	int64_t *tiles_at; /* [batch + 1]: the sequences' first tiles */
};

template <typename T, typename C>
hipError_t nvs_narrow(const nvs_kv &c, const nvs_kv_attend_args &a,
		      const nvs_plan &p, hipStream_t s);
template <typename T, typename C>
hipError_t nvs_wide(const nvs_kv &c, const nvs_kv_attend_args &a,
		    const nvs_plan &p, hipStream_t s);
template <typename T>
hipError_t nvs_join(const nvs_kv &c, const nvs_kv_attend_args &a,
		    const nvs_plan &p, bool narrow, hipStream_t s);

/* The keys [lo, hi) that some of the tokens [i0, i1] of s see, and their
 * tiles. */
struct key_range {
	int lo, hi;
	int first, last;
};

__device__ __forceinline__ key_range keys_of(const nvs_kv &c, int window,
					     const sequence &s, int i0, int i1,
					     int tile)
{
	const int64_t capacity = (int64_t)c.per_seq * c.page_size;
	const int64_t hi = min(s.pos + i1 + 1, capacity);
	const int64_t lo = window > 0 ? s.pos + i0 + 1 - window : 0;
	key_range k;

	k.lo = (int)min(max(lo, (int64_t)0), capacity);
	k.hi = (int)max(hi, (int64_t)0);
	if (k.hi <= k.lo)
		k.lo = k.hi = 0;
	k.first = k.lo / tile;
	k.last = (int)(((unsigned)k.hi + tile - 1) / tile);
	return k;
}

/* The wide kernel divides the tiles of a block of rows evenly between so
 * many parts. */
__device__ __forceinline__ int parts_of(const key_range &k, int most)
{
	return max(1, min(most, (k.last - k.first) / WIDE_LEAST));
}

/*
 * The narrow kernel lays the tiles of all its sequences end to end and
 * gives each of its blocks (for a cached head) the same number, however
 * unlike the sequences are: a block then has the end of one sequence, some
 * whole ones and the beginning of another, or a part of a long one.  Each
 * of its first and last pieces that is not a whole sequence goes to a slot
 * of the block's for the join.
 */
__device__ __forceinline__ key_range narrow_keys(const nvs_kv &c,
						 const nvs_kv_attend_args &a,
						 const nvs_plan &p,
						 const sequence &s, int tile)
{
	return keys_of(c, a.window, s, 0, s.count - 1, tile);
}

/* A sequence's tiles there: one at least where it has rows, as these have
 * a result; none where it is not for the narrow kernel or has more rows
 * than the caller said. */
__device__ __forceinline__ int narrow_tiles(const nvs_kv &c, const nvs_plan &p,
					    const sequence &s,
					    const key_range &k)
{
	const int64_t rows = (int64_t)s.count * (c.heads / c.kv_heads);

	return rows == 0 || rows > p.joined_rows ?
		       0 :
		       max(1, k.last - k.first);
}

/* How many blocks there are enough tiles for. */
__device__ __forceinline__ int64_t narrow_used(const nvs_plan &p,
					       int64_t tiles)
{
	return min((int64_t)p.narrow_blocks,
		   max(tiles / NARROW_LEAST, (int64_t)1));
}

/* The block that has tile x of `tiles`; block j of `used` begins with tile
 * j * tiles / used. */
__device__ __forceinline__ int narrow_block_of(int64_t x, int64_t tiles,
					       int64_t used)
{
	return (int)(((x + 1) * used - 1) / tiles);
}

__device__ __forceinline__ int64_t part_at(const nvs_plan &p, int kh,
					   int block, int slot)
{
	return (((int64_t)kh * p.narrow_blocks + block) * 2 + slot) * p.span;
}

struct share {
	int64_t from, to; /* tiles */
	int b;		  /* the sequence of tile `from`, or one before it */
	int64_t b_from;	  /* its first tile */
};

__device__ __forceinline__ share share_of(const nvs_kv &c,
					  const nvs_kv_attend_args &a,
					  const nvs_plan &p, int tile,
					  int block, bool leave)
{
	const int lane = threadIdx.x & 63;

	if (p.narrow_whole) {
		share m = {};

		if (block < c.batch) {
			const sequence s = sequence_of(c, block);

			m.b = block;
			m.to = uniform64(narrow_tiles(
				c, p, s, narrow_keys(c, a, p, s, tile)));
		}
		return m;
	}
	/* The tiles of sequence b0 + lane, and with those of the 63 before
	 * it: all the card's memory has fewer than 32 bits of them. */
	auto scan = [&](int b0, unsigned &own) {
		own = 0;
		if (b0 + lane < c.batch) {
			const sequence s = sequence_of(c, b0 + lane);

			own = narrow_tiles(c, p, s,
					   narrow_keys(c, a, p, s, tile));
		}
		unsigned sum = own;

		if (c.batch > 1)
#pragma unroll
			for (int o = 1; o < 64; o <<= 1) {
				const unsigned x = __shfl_up(sum, o);

				sum += lane >= o ? x : 0;
			}
		return sum;
	};
	int64_t tiles = 0;
	unsigned sum = 0, own = 0;

	for (int b0 = 0; b0 < c.batch; b0 += 64) {
		sum = scan(b0, own);
		if (leave && p.tiles_at && b0 + lane < c.batch)
			p.tiles_at[b0 + lane] = tiles + sum - own;
		tiles += (unsigned)__builtin_amdgcn_readlane(
			sum, c.batch > 1 ? 63 : 0);
	}
	if (leave && p.tiles_at && lane == 0)
		p.tiles_at[c.batch] = tiles;

	const int64_t used = narrow_used(p, tiles);
	share m = {};

	if (block >= used || tiles == 0)
		return m;
	m.from = block * tiles / used;
	m.to = (block + 1) * tiles / used;
	/* The last 64 sequences that begin no later, then the last one. */
	int64_t before = 0;

	for (int b0 = 0; c.batch > 1 && b0 < c.batch; b0 += 64) {
		if (c.batch > 64)
			sum = scan(b0, own);
		const int64_t all =
			(unsigned)__builtin_amdgcn_readlane(sum, 63);

		if (before + all > m.from) {
			const uint64_t later =
				__ballot(before + sum > m.from);
			const int n = __builtin_ctzll(later);

			m.b = b0 + n;
			m.b_from = before + (unsigned)__shfl(sum - own, n);
			break;
		}
		before += all;
	}
	m.from = uniform64(m.from);
	m.to = uniform64(m.to);
	m.b = uniform(m.b);
	m.b_from = uniform64(m.b_from);
	return m;
}

/* The number in its sequence of the page of a position. */
__device__ __forceinline__ int entry_of(const nvs_plan &p, int key)
{
	return (int)((unsigned)key * p.page_magic >> p.page_shift);
}

__device__ __forceinline__ int slot_of(const nvs_kv &c, const nvs_plan &p,
				       int key)
{
	return key - entry_of(p, key) * c.page_size;
}

/* The table's entry for a key in [lo, hi), -1 for other keys.  It is
 * looked up a tile ahead and not looked at before that tile's turn, which
 * would wait for it and for all loads before it. */
__device__ __forceinline__ int look_up(const nvs_plan &p, const int *table,
				       int key, const key_range &k)
{
	return key >= k.lo && key < k.hi ? table[entry_of(p, key)] : -1;
}

/* Whether an entry is a page of the cache. */
__device__ __forceinline__ bool is_page(const nvs_kv &c, int entry)
{
	return (unsigned)entry < (unsigned)c.pages;
}

/* Read in the place of keys and values that are none: a value that is not
 * seen still meets a weight of zero, so it has to be a finite number. */
static __device__ const u32x4 no_value[32] = {};

/* Where LDS memory lies, as the instructions count. */
__device__ __forceinline__ unsigned lds_at(const void *p)
{
	return (unsigned)(uintptr_t)(
		const __attribute__((address_space(3))) char *)p;
}

/*
 * 16 bytes (4) a lane from global memory to LDS, at `to` + 16 (4) * lane;
 * `to` is the same for the whole wave.  In assembly, because for the
 * builtin the compiler waits for all of a wave's loads before each read of
 * LDS, and the tile that is on its way would have to come before the
 * present one is read: the kernels wait by wait_loads() themselves.  There
 * is no result in a register, and m0 has its one wait state before it is
 * read.
 */
__device__ __forceinline__ void copy_to_lds(const char *from, unsigned to)
{
	asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\t"
		     "global_load_lds_dwordx4 %0, off"
		     :
		     : "v"(from), "s"(uniform(to))
		     : "memory", "m0");
}

__device__ __forceinline__ void copy4_to_lds(const int *from, unsigned to)
{
	asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\t"
		     "global_load_lds_dword %0, off"
		     :
		     : "v"(from), "s"(uniform(to))
		     : "memory", "m0");
}

/* Keeps the compiler from computing what is rarely wanted each time: a
 * branch that has this is a branch. */
__device__ __forceinline__ void rarely()
{
	asm volatile("");
}

/* Waits for a load here and not at each of its uses in a loop. */
__device__ __forceinline__ void arrived(u32x4 &x)
{
	asm volatile("" : "+v"(x));
}

/* At most N of the wave's loads still under way; no LDS access moves
 * across. */
template <int N> __device__ __forceinline__ void wait_loads()
{
	asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

__device__ __forceinline__ void wait_lds()
{
	asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}

/* Over the two halves (four quarters) of a wave. */
__device__ __forceinline__ f32x2 halves(float x)
{
	const unsigned u = __builtin_bit_cast(unsigned, x);
	const u32x2 r = __builtin_bit_cast(
		u32x2, __builtin_amdgcn_permlane32_swap(u, u, false, false));

	return __builtin_bit_cast(f32x2, r);
}

__device__ __forceinline__ f32x2 odd_even_quarters(float x)
{
	const unsigned u = __builtin_bit_cast(unsigned, x);
	const u32x2 r = __builtin_bit_cast(
		u32x2, __builtin_amdgcn_permlane16_swap(u, u, false, false));

	return __builtin_bit_cast(f32x2, r);
}

/*
 * A row's running softmax.  Weights are exp2(s * c - unit) with c =
 * scale * log2(e), unit = top * c - lift.  `top` follows the largest score
 * only once that is `lag` powers of two ahead, so that the results are
 * rescaled a few times and not with each tile; a weight then is at most
 * 2^(lift + lag), which both types hold, and the sum is made of the same
 * weights in 32 bits.
 */
template <typename T> struct softmax {
	float top = -INFINITY, sum = 0.f;

	__device__ __forceinline__ bool behind(float most, float c) const
	{
		return (most - top) * c > types<T>::lag ||
		       (top == -INFINITY && most > top);
	}

	/* Follow the maximum; what the results so far are multiplied by. */
	__device__ __forceinline__ float follow(float most, float c)
	{
		const float to = fmaxf(most, top);
		const float keep = top == -INFINITY ?
					   0.f :
					   __builtin_amdgcn_exp2f((top - to) *
								  c);
		top = to;
		sum *= keep;
		return keep;
	}

	__device__ __forceinline__ float unit(float c) const
	{
		return top == -INFINITY ? 0.f : top * c - types<T>::lift;
	}
};

/* Whether one of two numbers of type T (four e4m3) is infinite or NaN. */
template <typename C> __device__ __forceinline__ bool not_finite(unsigned w)
{
	if constexpr (sizeof(C) == 1)
		return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
	else
		return ((w & types<C>::exponent) + types<C>::one) &
		       0x80008000u;
}

/* A word of T (of e4m3) with zeros for what is infinite or NaN. */
template <typename C> __device__ __forceinline__ unsigned finite_only(unsigned w)
{
	constexpr int BITS = 8 * sizeof(C);
	constexpr unsigned FIELD = (1u << BITS) - 1u;

#pragma unroll
	for (int i = 0; i < 32; i += BITS)
		if (not_finite<C>(w & (FIELD << i)))
			w &= ~(FIELD << i);
	return w;
}

/* The factor of a row's scores, and what makes it positive, so that the
 * largest score has the largest weight: a sign to flip in the queries' bits,
 * or (zero) queries of zero. */
struct factor {
	float c;
	unsigned flip;
	bool zero;
};

__device__ __forceinline__ factor factor_of(float c)
{
	if (c == 0.f)
		return { 1.f, 0u, true };
	return { fabsf(c), c < 0.f ? 0x80008000u : 0u, false };
}

/* 0 times a word of T: NaN for what is infinite or NaN. */
template <typename T> __device__ __forceinline__ unsigned times_zero(unsigned w)
{
	return (not_finite<T>(w & 0xffffu) ? 0x7fffu : 0u) |
	       (not_finite<T>(w & 0xffff0000u) ? 0x7fff0000u : 0u);
}

/* The pieces of a row's queries, as its factor wants them. */
template <typename T, int N>
__device__ __forceinline__ void factored(const factor &f, u32x4 (&q)[N])
{
#pragma unroll
	for (int d = 0; d < N; d++)
		q[d] ^= f.flip;
	if (f.zero) {
		rarely();
#pragma unroll
		for (int d = 0; d < N; d++)
#pragma unroll
			for (int e = 0; e < 4; e++)
				q[d][e] = times_zero<T>(q[d][e]);
	}
}

/* x if it is infinite or NaN, else 0. */
__device__ __forceinline__ float odd_only(float x)
{
	return __builtin_isfinite(x) ? 0.f : x;
}

template <typename T>
__device__ __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 c)
{
	typedef typename types<T>::x8 x8;

	if constexpr (__is_same(T, bf16_t))
		return __builtin_amdgcn_mfma_f32_16x16x32_bf16(
			__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b),
			c, 0, 0, 0);
	else
		return __builtin_amdgcn_mfma_f32_16x16x32_f16(
			__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b),
			c, 0, 0, 0);
}

template <typename T>
__device__ __forceinline__ f32x16 mma32(u32x4 a, u32x4 b, f32x16 c)
{
	typedef typename types<T>::x8 x8;

	if constexpr (__is_same(T, bf16_t))
		return __builtin_amdgcn_mfma_f32_32x32x16_bf16(
			__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b),
			c, 0, 0, 0);
	else
		return __builtin_amdgcn_mfma_f32_32x32x16_f16(
			__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b),
			c, 0, 0, 0);
}

/* Four keys of one dimension a lane: of each 16 lanes, lane i gives the
 * address of 4 dimensions of key i / 4 and gets dimension i of 4 keys. */
__device__ __forceinline__ u32x2 read_keys4(const char *p)
{
	return __builtin_bit_cast(
		u32x2,
		__builtin_amdgcn_ds_read_tr16_b64_v4i16(
			(__attribute__((address_space(3))) s16x4 *)p));
}

/* The same of 8 keys in e4m3: lane i gives 8 dimensions of key i / 2. */
__device__ __forceinline__ u32x2 read_keys8(const char *p)
{
	typedef int s32x2 __attribute__((ext_vector_type(2)));

	return __builtin_bit_cast(
		u32x2,
		__builtin_amdgcn_ds_read_tr8_b64_v2i32(
			(__attribute__((address_space(3))) s32x2 *)p));
}

/* Rows that belong to no sequence: zeros where the buffer is the call's
 * own, and -inf in any case; by the launch's blocks `who` of `many`. */
template <typename T>
__device__ __forceinline__ void cover_padding(const nvs_kv &c,
					      const nvs_kv_attend_args &a,
					      int64_t who, int64_t many)
{
	if (!c.starts)
		return;
	const int *starts = c.starts;
	const int64_t head = max(0, min(starts[0], c.total));
	/* Sequences that pass the rows have none of them. */
	int64_t tail = starts[c.batch];

	if (tail > c.total)
		tail = starts[last_at_most(
			c.batch, c.total, [=](int i) {
				return (int64_t)starts[i];
			})];
	tail = max(head, min(tail, (int64_t)c.total));

	/* The rows before `head`, then those from `tail` on. */
	for (int64_t n = who; n < head + c.total - tail; n += many) {
		const int64_t row = n < head ? n : n - head + tail;

		for (int i = threadIdx.x; i < c.heads * c.dim / 8;
		     i += blockDim.x) {
			const int h = i / (c.dim / 8), d = i % (c.dim / 8) * 8;

			if (a.fill)
				*(u32x4 *)((T *)a.out + row * a.out_row +
					   h * a.out_head + d) = u32x4{};
			if (a.lse && d == 0)
				a.lse[row * c.heads + h] = -INFINITY;
		}
	}
}

#endif
