/*
 * nvshare-amd: attention of chunks of new tokens over a paged cache, and
 * the join of divided rows.  See kvattend.h for the division of the work.
 */
#include "kvattend.h"

namespace {

/*
 * Bound by the matrix and vector instructions: a wave's tile is 32 products
 * of 32x32x16 (1024 cycles) and 188 vector instructions, 32 of them
 * exponentials (870 cycles), which two waves of a SIMD overlap little: the
 * matrix units are busy 47 % of the time.
 *
 * Four waves of 32 rows share tiles of 64 keys and values in LDS, two of
 * each: while one is worked on, the next is on its way.  With rows of 128
 * two blocks fit a CU, and one computes while the other waits at its
 * barrier.  A 16-bit cache is loaded to LDS directly; e4m3 goes through
 * registers and lies in LDS as T, so that each value is widened once and
 * not by each wave.
 *
 * A chunk of 2048 tokens over 32049 keys (32 heads of 128, bfloat16): 1050
 * us, 990 TFLOP/s (1040 to 1114 on one card or another); four prompts of
 * 2048 from their first token: 171 us, 800.  Heads of 256: two chunks of
 * 1500 in a window of 1024, 75 us, 336; 256 + 212 registers leave one wave
 * a SIMD, and some 370 of a tile's 650 vector instructions move accumulators
 * between the two files.
 * Slower, for the chunk: tiles of 32 keys 1254 us, with three blocks a CU
 * 1647; blocks of 256 rows 1495; scores of the next tile made between the
 * exponentials of this one 1290 and more, as the registers run out.
 */
template <typename T, typename C, int D> struct wide {
	static constexpr int TILE = WIDE_TILE;
	static constexpr int RB = D * 2;	 /* bytes of a row in LDS */
	static constexpr int LR = RB / 16;	 /* lanes that load a row */
	static constexpr int RI = 64 / LR;	 /* rows of a load */
	static constexpr int NI = TILE / RI / 4; /* a wave's loads of a tile */
	static constexpr int BUFFER = TILE * RB;
	static constexpr int LDS = 4 * BUFFER;
	/* Waves of a SIMD: two blocks a CU, as far as LDS goes. */
	static constexpr int WAVES = LDS > 80 * 1024 ? 1 : 2;
	/* e4m3: 16-byte pieces of a thread. */
	static constexpr int NP = TILE * D / 16 / 256;

	/* Where a row's 16-byte pieces lie, so that reads of 16 rows (keys)
	 * and of 4 rows' 64 bytes (values) fall on all banks. */
	static __device__ __forceinline__ int turn_k(int row)
	{
		return RB >= 256 ? row & 15 : (row >> 1) & 7;
	}

	static __device__ __forceinline__ int turn_v(int row)
	{
		return RB >= 256 ? (row & 3) << 2 : ((row >> 1) & 1) << 2;
	}
};

template <typename T, typename C, int D>
__global__ __launch_bounds__(256, (wide<T, C, D>::WAVES)) void
wide_kernel(nvs_kv c, nvs_kv_attend_args a, nvs_plan p)
{
	typedef wide<T, C, D> W;
	constexpr int TILE = W::TILE, RB = W::RB, NI = W::NI;
	__shared__ __attribute__((aligned(16))) char lds[W::LDS];
	__shared__ int odd_tile[2];
	const int lane = threadIdx.x & 63;
	const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	const int col = lane & 31, half = lane >> 5;

	/* This block's sequence and rows: sequence b has the blocks from
	 * starts[b] * group / WIDE_ROWS + b on, which is room enough for
	 * its own.  The last blocks of rows, which see the most keys, go
	 * first. */
	const int group = c.heads / c.kv_heads;
	const int kh = blockIdx.x % c.kv_heads;
	const int part = blockIdx.x / c.kv_heads % p.wide_parts;
	const int at = p.wide_blocks - 1 -
		       blockIdx.x / c.kv_heads / p.wide_parts;
	int64_t block;
	int b;

	if (c.starts) {
		auto from = [&](int i) {
			return (int64_t)c.starts[i] * group / WIDE_ROWS + i;
		};
		if (from(0) > at)
			return;
		b = last_at_most(c.batch, at, from);
		if (b == c.batch)
			return;
		block = at - from(b);
	} else {
		b = at % c.batch;
		block = at / c.batch;
	}
	const sequence s = sequence_of(c, b);
	const int rows = s.count * group;

	if (block * WIDE_ROWS >= rows || rows <= p.narrow_rows)
		return;
	const int r0 = (int)block * WIDE_ROWS;
	const int i0 = r0 / group;
	const int i1 = min(s.count, (r0 + WIDE_ROWS - 1) / group + 1) - 1;
	key_range k = keys_of(c, a.window, s, i0, i1, TILE);
	const int parts = parts_of(k, p.wide_parts);
	const int per = (k.last - k.first + parts - 1) / parts;

	if (part >= parts)
		return;
	k.lo = uniform(k.lo);
	k.hi = uniform(k.hi);
	const int first = uniform(min(k.last, k.first + part * per));
	const int last = uniform(min(k.last, first + per));

	const int *const table = c.table + (int64_t)b * c.table_row;
	const float vs = sizeof(C) == 1 ? c.v_scale[kh] : 1.f;
	const factor f = factor_of(a.scale * 1.44269504f *
				   (sizeof(C) == 1 ? c.k_scale[kh] : 1.f));

	/* The lane's row, and the limits of the wave's. */
	const int r = r0 + wave * 32 + col;
	const bool real = r < rows;
	const int token = r / group, head = kh * group + r % group;
	auto limit = [&](int i) {
		return (int)max(min(s.pos + i, (int64_t)k.hi - 1),
				(int64_t)-1);
	};
	/* The row sees keys in (low, lim]. */
	const int lim = real ? limit(token) : -1;
	const int low = a.window > 0 ? (int)max(s.pos + token - a.window,
						(int64_t)-1) :
				       -1;
	const int w0 = min(rows - 1, r0 + wave * 32) / group;
	const int w1 = min(rows - 1, r0 + wave * 32 + 31) / group;
	const bool idle = r0 + wave * 32 >= rows;
	const int all = uniform(limit(w0)), most_lim = uniform(limit(w1));
	auto lowest = [&](int i) {
		return a.window > 0 ? uniform((int)max(
					      s.pos + i - a.window + 1,
					      (int64_t)0)) :
				      0;
	};
	const int any_low = lowest(w1), least_low = lowest(w0);
	/* Where the block's rows do not all see the same. */
	const int block_all = uniform(limit(i0)), block_low = lowest(i1);
	const bool alike = i0 == i1;

	u32x4 q[D / 16];
	const T *src = (const T *)a.q + (s.first + token) * a.q_row +
		       head * a.q_head;
#pragma unroll
	for (int d = 0; d < D / 16; d++) {
		q[d] = u32x4{};
		if (real)
			q[d] = *(const u32x4 *)(src + 16 * d + 8 * half);
	}
	factored<T>(f, q);

	softmax<T> sm;
	f32x16 out[D / 32];
#pragma unroll
	for (int d = 0; d < D / 32; d++)
#pragma unroll
		for (int e = 0; e < 16; e++)
			out[d][e] = 0.f;

	/* The page of key `lane` of a tile. */
	auto lookup = [&](int tile) {
		return tile < last ? look_up(p, table, tile * TILE + lane, k) :
				     -1;
	};
	/* Whether a tile lies in one page as a whole. */
	const bool one_page = c.page_size % TILE == 0 && p.near_slots;
	auto is_whole = [&](int pages) {
		return one_page && __all(is_page(c, pages));
	};
	constexpr int SIZE = sizeof(C);
	const char *const k_head = (const char *)c.k_cache +
				   kh * c.k_head * SIZE;
	const char *const v_head = (const char *)c.v_cache +
				   kh * c.v_head * SIZE;
	const unsigned k_step = (unsigned)(c.k_slot * SIZE);
	const unsigned v_step = (unsigned)(c.v_slot * SIZE);
	/* Where a tile that lies in one page begins. */
	auto tile_at = [&](const char *head, int64_t page_stride,
			   int64_t slot_stride, int key, int pages) {
		const int page = __builtin_amdgcn_readfirstlane(pages);

		return head + (page * page_stride +
			       slot_of(c, p, key) * slot_stride) *
				      SIZE;
	};
	/* Where a key's row begins; pages and slots are those of key `lane`
	 * of the tile. */
	auto row_at = [&](const char *head, int64_t page_stride,
			  int64_t slot_stride, int pages, int slots, int row) {
		const int page = __shfl(pages, row), slot = __shfl(slots, row);

		return !is_page(c, page) ?
			       (const char *)no_value :
			       head + (page * page_stride +
					  slot * slot_stride) *
						 SIZE;
	};
	/* 16 bits: request a tile for buffer n. */
	const int load_row = wave * NI * W::RI + lane / W::LR;
	const int load_piece = lane % W::LR;
	auto request = [&](int tile, int pages, int n) {
		const int key = tile * TILE;
		const unsigned to = lds_at(lds) + n * 2 * W::BUFFER +
				    wave * NI * 1024;

		if (is_whole(pages)) {
			const char *k = tile_at(k_head, c.k_page, c.k_slot,
						key, pages);
			const char *v = tile_at(v_head, c.v_page, c.v_slot,
						key, pages);
#pragma unroll
			for (int i = 0; i < NI; i++) {
				const int row = load_row + i * W::RI;

				copy_to_lds(k + (row * k_step +
						 (load_piece ^ W::turn_k(row)) *
							 16u),
					    to + i * 1024);
				copy_to_lds(v + (row * v_step +
						 (load_piece ^ W::turn_v(row)) *
							 16u),
					    to + W::BUFFER + i * 1024);
			}
			return;
		}
		const int slots = slot_of(c, p, key + lane);
#pragma unroll
		for (int i = 0; i < NI; i++) {
			rarely();
			const int row = load_row + i * W::RI;

			copy_to_lds(row_at(k_head, c.k_page, c.k_slot, pages,
					   slots, row) +
					    (load_piece ^ W::turn_k(row)) * 16,
				    to + i * 1024);
			copy_to_lds(row_at(v_head, c.v_page, c.v_slot, pages,
					   slots, row) +
					    (load_piece ^ W::turn_v(row)) * 16,
				    to + W::BUFFER + i * 1024);
		}
	};
	/* e4m3: fetch a tile into registers, put it into buffer n. */
	u32x4 hold[2][SIZE == 1 ? W::NP : 1];
	auto fetch = [&](int tile, int pages) {
		const int key = tile * TILE;
		const bool whole = is_whole(pages);
		const int slots = slot_of(c, p, key + lane);
		const char *k = nullptr, *v = nullptr;

		if (whole) {
			k = tile_at(k_head, c.k_page, c.k_slot, key, pages);
			v = tile_at(v_head, c.v_page, c.v_slot, key, pages);
		}
#pragma unroll
		for (int i = 0; i < W::NP; i++) {
			const int n = i * 256 + threadIdx.x;
			const int row = n / (D / 16), piece = n % (D / 16);
			const char *from_k, *from_v;

			if (whole) {
				from_k = k + row * k_step;
				from_v = v + row * v_step;
			} else {
				rarely();
				from_k = row_at(k_head, c.k_page, c.k_slot,
						pages, slots, row);
				from_v = row_at(v_head, c.v_page, c.v_slot,
						pages, slots, row);
			}
			hold[0][i] = *(const u32x4 *)(from_k + piece * 16);
			hold[1][i] = *(const u32x4 *)(from_v + piece * 16);
		}
	};
	auto put = [&](int n) {
		char *to = lds + n * 2 * W::BUFFER;
#pragma unroll
		for (int i = 0; i < W::NP; i++) {
			const int m = i * 256 + threadIdx.x;
			const int row = m / (D / 16), piece = m % (D / 16) * 2;
#pragma unroll
			for (int e = 0; e < 2; e++) {
				const u32x4 w = hold[0][i], x = hold[1][i];

				*(u32x4 *)(to + row * RB +
					   ((piece + e) ^ W::turn_k(row)) *
						   16) =
					widen8<T>(u32x2{ w[2 * e],
							 w[2 * e + 1] });
				*(u32x4 *)(to + W::BUFFER + row * RB +
					   ((piece + e) ^ W::turn_v(row)) *
						   16) =
					widen8<T>(u32x2{ x[2 * e],
							 x[2 * e + 1] });
			}
		}
	};

	int pages = lookup(first), next = lookup(first + 1);

	if (first < last) {
		if constexpr (SIZE == 2) {
			request(first, pages, 0);
		} else {
			fetch(first, pages);
			put(0);
		}
	}
#pragma unroll
	for (int d = 0; d < D / 16; d++)
		arrived(q[d]);
	for (int t = first; t < last; t++) {
		const int n = (t - first) & 1;
		const char *const k_lds = lds + n * 2 * W::BUFFER;
		char *const v_lds = lds + n * 2 * W::BUFFER + W::BUFFER;
		const uint64_t valid = __ballot(is_page(c, pages));
		const int key0 = t * TILE;

		/* This tile has come, and all are done with the other. */
		if constexpr (SIZE == 2)
			wait_loads<0>();
		wait_lds();
		__builtin_amdgcn_s_barrier();
		asm volatile("" ::: "memory");
		if (t + 1 < last) {
			if constexpr (SIZE == 2)
				request(t + 1, next, n ^ 1);
			else
				fetch(t + 1, next);
		}
		pages = next;
		next = lookup(t + 2);

		/* 0 * inf is no number: values that are not finite and not
		 * seen by all rows are added for those that see them, and
		 * the product takes zeros in their place. */
		const bool uneven = !alike && (key0 + TILE - 1 > block_all ||
					       key0 < block_low);
		if (uneven) {
			bool odd = false;

			if (threadIdx.x == 0)
				odd_tile[n] = 0;
			__syncthreads();
			for (int i = 0; i < NI; i++) {
				const u32x4 w = *(
					const u32x4 *)(v_lds +
						       (wave * NI + i) * 1024 +
						       lane * 16);

				odd |= not_finite<T>(w[0]) |
				       not_finite<T>(w[1]) |
				       not_finite<T>(w[2]) | not_finite<T>(w[3]);
			}
			if (odd)
				odd_tile[n] = 1;
			__syncthreads();
			if (odd_tile[n]) {
#pragma unroll 1
				for (int j = 0; j < TILE; j++) {
					const int key = key0 + j;
					const bool sees =
						(valid >> j & 1) &&
						key <= lim && key > low;
#pragma unroll
					for (int d = 0; d < D / 8; d++) {
						const char *from =
							v_lds + j * RB +
							(d ^ W::turn_v(j)) *
								16 +
							half * 8;
						asm volatile("" ::: "memory");
						const u32x2 w =
							*(const u32x2 *)from;
						const T *v = (const T *)&w;
#pragma unroll
						for (int e = 0; e < 4; e++)
							out[d / 4][d % 4 * 4 +
								   e] +=
								sees ? odd_only((
									       float)v[e]) :
								       0.f;
					}
				}
				__syncthreads();
#pragma unroll 1
				for (int i = 0; i < NI; i++) {
					u32x4 *to = (u32x4 *)(v_lds +
							      (wave * NI + i) *
								      1024 +
							      lane * 16);
					u32x4 w = *to;

#pragma unroll
					for (int e = 0; e < 4; e++)
						w[e] = finite_only<T>(w[e]);
					*to = w;
				}
				__syncthreads();
			}
		}

		if (!idle && key0 <= most_lim && key0 > least_low - TILE) {
			/* Keys: S^T = K Q^T. */
			f32x16 score[2];
#pragma unroll
			for (int h = 0; h < 2; h++)
#pragma unroll
				for (int e = 0; e < 16; e++)
					score[h][e] = 0.f;
#pragma unroll
			for (int d = 0; d < D / 16; d++)
#pragma unroll
				for (int h = 0; h < 2; h++) {
					const int row = 32 * h + col;
					const u32x4 w = *(
						const u32x4 *)(k_lds +
							       row * RB +
							       ((2 * d + half) ^
								W::turn_k(
									row)) *
								       16);

					score[h] = mma32<T>(w, q[d], score[h]);
				}
			/* Weights. */
			if (valid != ~0ull || key0 + TILE - 1 > all ||
			    key0 < any_low) {
				rarely();
				/* As seen from the lane's first key. */
				const uint64_t mine = valid >> 4 * half;
				const int to = lim - key0 - 4 * half;
				const int after = low - key0 - 4 * half;
#pragma unroll
				for (int h = 0; h < 2; h++)
#pragma unroll
					for (int e = 0; e < 16; e++) {
						const int j = 32 * h +
							      8 * (e >> 2) +
							      (e & 3);
						const bool sees =
							(mine >> j & 1) &
							(j <= to) & (j > after);

						score[h][e] = sees ?
								      score[h][e] :
								      -INFINITY;
					}
			}
			float most = score[0][0];
#pragma unroll
			for (int e = 1; e < 16; e++)
				most = fmaxf(most, score[0][e]);
#pragma unroll
			for (int e = 0; e < 16; e++)
				most = fmaxf(most, score[1][e]);
			const f32x2 y = halves(most);

			most = fmaxf(y[0], y[1]);
			if (__any(sm.behind(most, f.c))) {
				const float keep = sm.follow(most, f.c);
#pragma unroll
				for (int d = 0; d < D / 32; d++)
					out[d] *= keep;
			}
			const float unit = sm.unit(f.c);
			/* Weights are rounded once to T before they meet the
			 * values; their sum is made of the unrounded ones.
			 * With the results' own rounding that is 2.4e-3 of
			 * their size in bfloat16, 2.9e-4 in float16, where
			 * two parts of T, as the narrow kernel has, leave
			 * 1.7e-3 and 2.1e-4 and half as many products again:
			 * 1385 us instead of 1054 (the chunk above), 484
			 * instead of 394 (ragged prompts of up to 4096). */
			u32x4 weight[4];
#pragma unroll
			for (int h = 0; h < 2; h++) {
#pragma unroll
				for (int e = 0; e < 16; e++) {
					score[h][e] = __builtin_amdgcn_exp2f(
						__builtin_fmaf(score[h][e],
							       f.c, -unit));
					sm.sum += score[h][e];
				}
#pragma unroll
				for (int e = 0; e < 8; e++)
					weight[2 * h + e / 4][e % 4] =
						pack2<T>(score[h][2 * e],
							 score[h][2 * e + 1]);
			}

			/* Values: O^T += V^T P^T. */
#pragma unroll
			for (int h = 0; h < 4; h++) {
				const int row = 16 * h + 4 * half +
						((lane & 15) >> 2);
#pragma unroll
				for (int d = 0; d < D / 32; d++) {
					const int piece =
						(4 * d + 2 * (lane >> 4 & 1) +
						 ((lane & 3) >> 1)) ^
						W::turn_v(row);
					const char *from = v_lds + row * RB +
							   piece * 16 +
							   (lane & 1) * 8;
					const u32x2 lo = read_keys4(from);
					const u32x2 hi =
						read_keys4(from + 8 * RB);

					out[d] = mma32<T>(u32x4{ lo[0], lo[1],
								 hi[0],
								 hi[1] },
							  weight[h], out[d]);
				}
			}
		}
		if constexpr (SIZE == 1)
			if (t + 1 < last)
				put(n ^ 1);
	}

	/* The result: lane `col` of each half has 4 of each 8 dimensions. */
	const f32x2 y = halves(sm.sum);
	const float sum = y[0] + y[1];
	const int64_t row = s.first + token;
	const float unit = sm.top == -INFINITY ? -INFINITY : sm.unit(f.c);

	if (!real)
		return;
	if (parts > 1) {
		const int64_t at_row =
			(part * (int64_t)c.total + row) * c.heads + head;
#pragma unroll
		for (int d = 0; d < D / 8; d++) {
			const f32x16 x = out[d / 4];
			const int e = d % 4 * 4;

			*(f32x4 *)(p.wide_out + at_row * D + 8 * d +
				   4 * half) =
				f32x4{ x[e], x[e + 1], x[e + 2], x[e + 3] };
		}
		if (half == 0)
			p.wide_sum[at_row] = f32x2{ unit, sum };
		return;
	}
	const float inv = sum == 0.f ? 0.f : vs / sum;
#pragma unroll
	for (int d = 0; d < D / 8; d++) {
		const f32x16 x = out[d / 4];
		const int e = d % 4 * 4;
		const u32x2 w = { pack2<T>(x[e] * inv, x[e + 1] * inv),
				  pack2<T>(x[e + 2] * inv, x[e + 3] * inv) };

		*(u32x2 *)((T *)a.out + row * a.out_row + head * a.out_head +
			   8 * d + 4 * half) = w;
	}
	if (a.lse && half == 0)
		a.lse[row * c.heads + head] =
			sum == 0.f ? -INFINITY :
				     (unit + __builtin_amdgcn_logf(sum)) *
					     0.693147181f;
}

/*
 * Join the parts of rows whose keys were divided.  Rows with one part have
 * their result already.  A row has WAVES waves, each of them with every
 * WAVES-th part, several at a time so that their loads are under way
 * together.
 */
template <typename T, int D, bool NARROW, int WAVES>
__global__ __launch_bounds__(256) void join_kernel(nvs_kv c,
						   nvs_kv_attend_args a,
						   nvs_plan p, int all_rows)
{
	constexpr int PER = D / 64; /* dimensions of a lane */
	constexpr int MANY = WAVES > 1 ? 8 : 4; /* parts at a time */
	typedef float vec __attribute__((ext_vector_type(PER)));
	__shared__ vec add[4][64];
	__shared__ float units[4], sums[4];
	const int lane = threadIdx.x % 64;
	const int wave = uniform(threadIdx.x / 64);
	const int group = c.heads / c.kv_heads;
	const int index = (blockIdx.x * 4 + wave) / WAVES;
	const int tp = wave % WAVES;
	int b = 0, r = 0, head = 0, parts = 1;
	sequence s = {};
	/* Where part n is: the first at at0, the others at + n * step. */
	int64_t at0 = 0, at = 0, step = 0;

	if (NARROW && index < all_rows) {
		const int item = index / p.joined_rows, kh = item % c.kv_heads;

		b = item / c.kv_heads;
		r = index % p.joined_rows;
		head = kh * group + r % group;
		const int64_t from = p.tiles_at[b], to = p.tiles_at[b + 1];
		const int64_t tiles = p.tiles_at[c.batch];

		s = sequence_of(c, b);
		if (from < to && r < s.count * group) {
			const int64_t used = narrow_used(p, tiles);
			const int j = narrow_block_of(from, tiles, used);

			parts = narrow_block_of(to - 1, tiles, used) - j + 1;
			at = part_at(p, kh, j, 0) + r;
			step = 2 * p.span;
			/* Not the first piece of its block: the other slot. */
			at0 = from > j * tiles / used ? at + p.span : at;
		}
	} else if (index < all_rows) {
		head = index % c.heads;
		b = sequence_at(c, index / c.heads);
		if (b >= 0) {
			s = sequence_of(c, b);
			const int rows = s.count * group;

			r = (index / c.heads - s.first) * group + head % group;
			if (r < rows && rows > p.narrow_rows) {
				const int r0 = r / WIDE_ROWS * WIDE_ROWS;

				parts = parts_of(
					keys_of(c, a.window, s, r0 / group,
						min(s.count,
						    (r0 + WIDE_ROWS - 1) /
								    group +
							    1) -
							1,
						WIDE_TILE),
					p.wide_parts);
			}
		}
		at = at0 = index;
		step = (int64_t)c.total * c.heads;
	}
	parts = uniform(parts);
	if (parts < 2)
		return; /* with WAVES = 4 the whole block */
	const f32x2 *const part_sum = NARROW ? p.narrow_sum : p.wide_sum;
	const float *const part_out = (NARROW ? p.narrow_out : p.wide_out) +
				      PER * lane;
	float unit = -INFINITY, sum = 0.f;
	vec x = {};
	auto weigh = [](float u, float top) {
		return u == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(u - top);
	};

	for (int n0 = tp; n0 < parts; n0 += MANY * WAVES) {
		f32x2 y[MANY];
		vec v[MANY];
		float top = unit;

#pragma unroll
		for (int i = 0; i < MANY; i++) {
			const int n = n0 + i * WAVES;
			const int m = min(n, parts - 1);
			const int64_t place = m ? at + m * step : at0;

			y[i] = part_sum[place];
			v[i] = *(const vec *)(part_out + place * D);
			/* Beyond the parts: nothing, and not a part with
			 * weight 0, which makes NaN of its infinities. */
			if (n >= parts) {
				y[i] = f32x2{ -INFINITY, 0.f };
				v[i] = vec{};
			}
		}
#pragma unroll
		for (int i = 0; i < MANY; i++)
			top = fmaxf(top, y[i][0]);
		const float keep = weigh(unit, top);

		sum *= keep;
		x *= keep;
#pragma unroll
		for (int i = 0; i < MANY; i++) {
			const float m = weigh(y[i][0], top);

			/* A part that saw no key has weight 0 and zeros, one
			 * whose scores are NaN weight 0 and NaN. */
			sum += m * y[i][1];
			x += m * v[i];
		}
		unit = top;
	}
	if (WAVES > 1) {
		add[wave][lane] = x;
		if (lane == 0) {
			units[wave] = unit;
			sums[wave] = sum;
		}
		__syncthreads();
		if (tp)
			return;
		float top = unit;

		for (int n = 1; n < WAVES; n++)
			top = fmaxf(top, units[n]);
		const float keep = weigh(unit, top);

		sum *= keep;
		x *= keep;
		for (int n = 1; n < WAVES; n++) {
			const float m = weigh(units[n], top);

			sum += m * sums[n];
			x += m * add[n][lane];
		}
		unit = top;
	}
	const int kh = head / group;
	const float inv =
		sum == 0.f ? 0.f : (c.v_scale ? c.v_scale[kh] : 1.f) / sum;
	const int64_t row = s.first + r / group;
	T *o = (T *)a.out + row * a.out_row + head * a.out_head + PER * lane;

	if constexpr (PER == 1)
		*o = (T)(x[0] * inv);
	else
#pragma unroll
		for (int e = 0; e < PER; e += 2)
			*(unsigned *)(o + e) =
				pack2<T>(x[e] * inv, x[e + 1] * inv);
	if (a.lse && lane == 0)
		a.lse[row * c.heads + head] =
			sum == 0.f ? -INFINITY :
				     (unit + __builtin_amdgcn_logf(sum)) *
					     0.693147181f;
}

template <typename T, int D, bool NARROW>
void join(const nvs_kv &c, const nvs_kv_attend_args &a, const nvs_plan &p,
	  hipStream_t s)
{
	const int rows = NARROW ? c.batch * c.kv_heads * p.joined_rows :
				  c.total * c.heads;
	/* Many parts (64 of each of 32 rows, one sequence over 120001 keys)
	 * are read by a block, 5.5 us where a wave took 16; few (2048 rows,
	 * a batch of 64) by a wave, 5 us where a block took 9. */
	const int64_t parts = NARROW ? p.narrow_blocks / c.batch :
				       p.wide_parts;

	if (parts >= 16)
		hipLaunchKernelGGL((join_kernel<T, D, NARROW, 4>),
				   dim3(rows), dim3(256), 0, s, c, a, p, rows);
	else
		hipLaunchKernelGGL((join_kernel<T, D, NARROW, 1>),
				   dim3((rows + 3) / 4), dim3(256), 0, s, c, a,
				   p, rows);
}

} /* namespace */

template <typename T, typename C>
hipError_t nvs_wide(const nvs_kv &c, const nvs_kv_attend_args &a,
		    const nvs_plan &p, hipStream_t s)
{
	const dim3 grid(p.wide_blocks * c.kv_heads * p.wide_parts);

	if (c.dim == 64)
		hipLaunchKernelGGL((wide_kernel<T, C, 64>), grid, dim3(256), 0,
				   s, c, a, p);
	else if (c.dim == 128)
		hipLaunchKernelGGL((wide_kernel<T, C, 128>), grid, dim3(256),
				   0, s, c, a, p);
	else
		hipLaunchKernelGGL((wide_kernel<T, C, 256>), grid, dim3(256),
				   0, s, c, a, p);
	return hipGetLastError();
}

template <typename T>
hipError_t nvs_join(const nvs_kv &c, const nvs_kv_attend_args &a,
		    const nvs_plan &p, bool narrow, hipStream_t s)
{
	if (c.dim == 64)
		narrow ? join<T, 64, true>(c, a, p, s) :
			 join<T, 64, false>(c, a, p, s);
	else if (c.dim == 128)
		narrow ? join<T, 128, true>(c, a, p, s) :
			 join<T, 128, false>(c, a, p, s);
	else
		narrow ? join<T, 256, true>(c, a, p, s) :
			 join<T, 256, false>(c, a, p, s);
	return hipGetLastError();
}

#define INSTANCE(T, C)                                                     \
	template hipError_t nvs_wide<T, C>(const nvs_kv &,                 \
					   const nvs_kv_attend_args &,     \
					   const nvs_plan &,               \
					   hipStream_t);
INSTANCE(bf16_t, bf16_t)
INSTANCE(bf16_t, e4m3_t)
INSTANCE(fp16_t, fp16_t)
INSTANCE(fp16_t, e4m3_t)
#define INSTANCE_JOIN(T)                                                   \
	template hipError_t nvs_join<T>(const nvs_kv &,                    \
					const nvs_kv_attend_args &,        \
					const nvs_plan &, bool,            \
					hipStream_t);
INSTANCE_JOIN(bf16_t)
INSTANCE_JOIN(fp16_t)
