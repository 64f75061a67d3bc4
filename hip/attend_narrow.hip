/*
 * nvshare-amd: attention of a few rows (single tokens, drafts) over a
 * paged cache.  See kvattend.h for the division of the work.
 */
#include "kvattend.h"

namespace {

/*
 * Bound by the cache's bytes: 4 D operations for 2 D * 2 bytes of a key and
 * value, times the few rows that see them.
 *
 * A block has W waves and NC columns of 16 rows, all in every wave; wave w
 * takes each W-th tile of its block's keys.  A wave's tiles lie in LDS of
 * its own, filled by direct loads, so the waves never wait for each other:
 * the next tile's keys are requested as soon as this one's are read, its
 * values as soon as this one's are, and the loads of 8 waves a CU (16 with
 * the smallest rows) are under way together, up to 128 KiB of them.  What
 * the waves have is added up in LDS at the end.  Products of 16 columns
 * take half the registers and exponentials of those of 32 and lose nothing,
 * as a block seldom has more rows.
 *
 * A tile has 32 keys, 64 where 32 would be less than 8 KiB: what is done
 * once a tile (its page, its mask, the maximum over the lanes) would take
 * longer than its loads.
 *
 * One token over 120001 keys (8 cached heads of 128, bfloat16, 492 MB): 91
 * us, 5.4 TB/s; 64 tokens over up to 16384 keys each (2.36 GB): 431 us, 5.5
 * TB/s (423 without any arithmetic; plain loads of the same pages reach 6.0
 * to 6.2 TB/s).  e4m3 (1.10 GB, rows of 128 bytes): 230 us, 4.8 TB/s.  17
 * to 32 rows with heads of 256 spill 48 registers (27 with e4m3): 8 x 8
 * tokens over 5000 keys 128 us where 8 x 4 take 71.
 */
template <typename T, typename C, int D, int NC, int W> struct narrow {
	static constexpr int RB = D * sizeof(C); /* bytes of a row in LDS */
	static constexpr int TILE = nvs_narrow_tile(D, sizeof(C));
	static constexpr int LR = RB / 16;  /* lanes that load a row */
	static constexpr int RI = 64 / LR;  /* rows of a load */
	static constexpr int NI = TILE / RI; /* loads of a tile */
	static constexpr int STAGE = W * 2 * TILE * RB;
	static constexpr int OUT_ROW = D + 4; /* floats, off the banks */
	static constexpr int MERGE = W * 16 * NC * OUT_ROW * 4;
	static constexpr int LDS = STAGE > MERGE ? STAGE : MERGE;
	/* Waves that a SIMD holds: as LDS allows, and with 32 rows as the
	 * registers do. */
	static constexpr int WAVES = LDS > 76 * 1024 || W == 2	   ? 1 :
				     LDS <= 38 * 1024 && NC == 1 ? 4 :
								     2;

	/* Where a row's 16-byte pieces lie: turned about so that the 16
	 * rows of a read fall on all banks. */
	static __device__ __forceinline__ int turn_k(int row)
	{
		return RB >= 256 ? row & 15 :
		       RB == 128 ? (row >> 1) & 7 :
				   (row >> 2) & 3;
	}

	static __device__ __forceinline__ int turn_v(int row)
	{
		if (sizeof(C) == 2)
			return RB >= 256 ? (row & 7) << 1 :
					   ((row >> 1) & 3) << 1;
		return RB == 256 ? (row & 7) | (row >> 4 & 1) << 3 :
		       RB == 128 ? (row >> 1 & 3) | (row >> 4 & 1) << 2 :
				   (row >> 2 & 1) | (row >> 4 & 1) << 1;
	}
};

template <typename T, typename C, int D, int NC, int W>
__global__ __launch_bounds__(64 * W, (narrow<T, C, D, NC, W>::WAVES)) void
narrow_kernel(nvs_kv c, nvs_kv_attend_args a, nvs_plan p)
{
	typedef narrow<T, C, D, NC, W> N;
	constexpr int TILE = N::TILE, RB = N::RB, NI = N::NI;
	constexpr int SUBS = TILE / 32;
	__shared__ __attribute__((aligned(16))) char lds[N::LDS];
	__shared__ int entries[W][2][64];
	__shared__ float tops[W][16 * NC], sums[W][16 * NC];
	const int lane = threadIdx.x & 63;
	const int wave = uniform(threadIdx.x >> 6);
	const int col = lane & 15, quarter = lane >> 4;
	const int group = c.heads / c.kv_heads;

	/* With 8 cached heads each has an XCD of its own.  (All heads of the
	 * same keys on one XCD: 399 us where this takes 383, for 64 tokens
	 * over 8192 keys each.) */
	const int kh = blockIdx.x % c.kv_heads;
	const int block = blockIdx.x / c.kv_heads;

	/* With starts there is always a narrow launch. */
	cover_padding<T>(c, a, blockIdx.x, gridDim.x);

	char *const k_lds = lds + wave * 2 * TILE * RB;
	char *const v_lds = k_lds + TILE * RB;
	const unsigned k_at = lds_at(lds) + wave * 2 * TILE * RB;
	const unsigned v_at = k_at + TILE * RB;
	const float vs = sizeof(C) == 1 ? c.v_scale[kh] : 1.f;
	const factor f = factor_of(a.scale * 1.44269504f *
				   (sizeof(C) == 1 ? c.k_scale[kh] : 1.f));
	/* Which 16 bytes of a tile's rows this lane loads. */
	const int lr = lane / N::LR, lc = lane % N::LR;

	/* This block's share of all sequences' tiles, one after the other;
	 * block 0 leaves where each begins for the join. */
	const share mine = share_of(c, a, p, TILE, block,
				    blockIdx.x == 0 && wave == 0);
	int64_t at = mine.from; /* the next tile */
	int b = mine.b, odd_b = block, odd_r0 = 0;
	int64_t b_from = mine.b_from; /* the first tile of sequence b */

	for (;;) {
		/* The next piece: rows r0 and on of sequence b, its tiles
		 * [first, last), and where its result goes. */
		sequence s;
		key_range k;
		int r0 = 0, first, last, slot = -1;

		if (at < mine.to && b < c.batch) {
			s = sequence_of(c, b);
			k = narrow_keys(c, a, p, s, TILE);
			const int64_t b_to = b_from + narrow_tiles(c, p, s, k);

			if (b_to <= at) {
				b_from = b_to;
				b++;
				continue;
			}
			const int64_t to = min(b_to, mine.to);

			first = k.first + (int)(at - b_from);
			last = min(k.first + (int)(to - b_from), k.last);
			if (at > b_from || to < b_to)
				slot = at == mine.from ? 0 : 1;
			at = to;
		} else {
			/* Sequences with more rows than the caller said:
			 * undivided, so many rows at a time. */
			if (!c.starts || p.narrow_rows < 0x7fffffff ||
			    odd_b >= c.batch)
				break;
			b = odd_b;
			s = sequence_of(c, b);
			if (s.count * group <= p.joined_rows ||
			    odd_r0 >= s.count * group) {
				odd_b += p.narrow_blocks;
				odd_r0 = 0;
				continue;
			}
			r0 = odd_r0;
			odd_r0 += 16 * NC;
			k = keys_of(c, a.window, s, r0 / group,
				    min(s.count,
					(r0 + 16 * NC - 1) / group + 1) -
					    1,
				    TILE);
			first = k.first;
			last = k.last;
		}
		first = uniform(first);
		last = uniform(last);
		k.lo = uniform(k.lo);
		k.hi = uniform(k.hi);
		const int rows = s.count * group;
		const int i0 = r0 / group;
		const int i1 = min(s.count, (r0 + 16 * NC - 1) / group + 1) -
			       1;
		const int *const table = c.table + (int64_t)b * c.table_row;

		u32x4 q[NC][D / 32];
		/* The lane's row sees keys in (low, lim]. */
		int lim[NC], low[NC];
#pragma unroll
		for (int n = 0; n < NC; n++) {
			const int r = r0 + 16 * n + col;
			const int i = r / group;

			lim[n] = low[n] = -1;
			if (r < rows) {
				const T *src = (const T *)a.q +
					       (s.first + i) * a.q_row +
					       (kh * group + r % group) *
						       a.q_head;
				lim[n] = (int)max(min(s.pos + i,
						      (int64_t)k.hi - 1),
						  (int64_t)-1);
				if (a.window > 0)
					low[n] = (int)max(s.pos + i - a.window,
							  (int64_t)-1);
#pragma unroll
				for (int d = 0; d < D / 32; d++)
					q[n][d] = *(const u32x4 *)(src +
								   32 * d +
								   8 * quarter);
				factored<T>(f, q[n]);
			} else {
#pragma unroll
				for (int d = 0; d < D / 32; d++)
					q[n][d] = u32x4{};
			}
		}
		/* The limits of all rows: keys up to `all` are seen by each
		 * unless a window ends before. */
		const int all = uniform((int)min(max(s.pos + i0, (int64_t)-1),
						 (int64_t)k.hi - 1));
		const int any_low =
			a.window > 0 ? uniform((int)max(s.pos + i1 -
								a.window + 1,
							(int64_t)0)) :
				       0;
		const bool alike = s.pos + i0 == s.pos + i1;

		/* Not before the first tile is on its way. */
		auto queries_arrived = [&]() {
#pragma unroll
			for (int n = 0; n < NC; n++)
#pragma unroll
				for (int d = 0; d < D / 32; d++)
					arrived(q[n][d]);
		};

		softmax<T> sm[NC];
		f32x4 out[NC][D / 16];
#pragma unroll
		for (int n = 0; n < NC; n++)
#pragma unroll
			for (int d = 0; d < D / 16; d++)
				out[n][d] = f32x4{};

		/* Request a tile's rows.  `pages` has the page of key lane %
		 * TILE of the tile; whole: all are in the same.  Addresses
		 * are made anew each time: kept ones would take more
		 * registers than the results. */
		constexpr int SIZE = sizeof(C);
		auto request = [&](const void *cache, int64_t page_stride,
				   int64_t slot_stride, int64_t head, int tile,
				   int pages, bool whole, bool values,
				   unsigned to) {
			const int key = tile * TILE;
			const char *from = (const char *)cache +
					   kh * head * SIZE;
			int r = lr;

			if (whole) {
				const int page =
					__builtin_amdgcn_readfirstlane(pages);
				const unsigned step =
					(unsigned)(slot_stride * SIZE);

				from += (page * page_stride +
					 slot_of(c, p, key) * slot_stride) *
					SIZE;
#pragma unroll
				for (int i = 0; i < NI; i++) {
					asm volatile("" : "+v"(r));
					const int row = i * N::RI + r;
					const unsigned piece =
						lc ^ (values ? N::turn_v(row) :
							       N::turn_k(row));

					copy_to_lds(from + (row * step +
							    piece * 16),
						    to + i * 1024);
				}
				return;
			}
			const int slots =
				slot_of(c, p, key + (lane & (TILE - 1)));
#pragma unroll
			for (int i = 0; i < NI; i++) {
				asm volatile("" : "+v"(r));
				const int row = i * N::RI + r;
				const int piece = lc ^ (values ?
								N::turn_v(row) :
								N::turn_k(row));
				const int page = __shfl(pages, row);
				const int slot = __shfl(slots, row);
				const char *at =
					from + (page * page_stride +
						slot * slot_stride) *
						       SIZE;

				if (page < 0)
					at = (const char *)no_value;
				copy_to_lds(at + piece * 16, to + i * 1024);
			}
		};
		const bool one_page = c.page_size % TILE == 0 && p.near_slots;
		auto is_whole = [&](int pages) {
			return one_page && __all(pages >= 0);
		};
		/* Key lane % TILE of a tile; below zero where one beyond the
		 * last passes 31 bits. */
		auto key_of = [&](int tile) {
			return (int)((unsigned)tile * TILE +
				     (lane & (TILE - 1)));
		};
		/* The table's entry for it, or the nearest one that some row
		 * sees. */
		auto entry = [&](int tile) {
			const int key = key_of(tile);

			return table + entry_of(p, min(max(key, k.lo),
						       k.hi - 1));
		};
		/* The pages, -1 for keys that no row sees. */
		auto pages_of = [&](int tile, int entry) {
			const int key = key_of(tile);

			return key >= k.lo && key < k.hi && is_page(c, entry) ?
				       entry :
				       -1;
		};

		/* On their way at the loop's head, in this order: the table's
		 * entries for the next tile, this one's keys, its values. */
		int t = first + wave, turn = 0;
		int pages = -1;
		bool whole = false;

		if (t < last) {
			pages = pages_of(t, *entry(t));
			whole = is_whole(pages);
			copy4_to_lds(entry(t + W), lds_at(entries[wave][0]));
			request(c.k_cache, c.k_page, c.k_slot, c.k_head, t,
				pages, whole, false, k_at);
			request(c.v_cache, c.v_page, c.v_slot, c.v_head, t,
				pages, whole, true, v_at);
		}
		queries_arrived();
		for (; t < last; t += W, turn ^= 1) {
			const uint64_t valid = __ballot(pages >= 0);
			const bool more = t + W < last;
			const int key0 = t * TILE;

			wait_loads<NI>();
			const int pages1 =
				pages_of(t + W, entries[wave][turn][lane]);
			const bool whole1 = is_whole(pages1);

			/* Keys: S^T = K Q^T. */
			wait_loads<NI>();
			f32x4 score[NC][2 * SUBS];
#pragma unroll
			for (int h = 0; h < 2 * SUBS; h++) {
#pragma unroll
				for (int n = 0; n < NC; n++)
					score[n][h] = f32x4{};
#pragma unroll
				for (int d = 0; d < D / 32; d++) {
					const int row = 16 * h + col;
					u32x4 w;

					if constexpr (sizeof(C) == 2) {
						const int piece =
							(4 * d + quarter) ^
							N::turn_k(row);

						w = *(const u32x4
							      *)(k_lds +
								 row * RB +
								 piece * 16);
					} else {
						const int piece =
							(2 * d +
							 (quarter >> 1)) ^
							N::turn_k(row);

						w = widen8<T>(
							*(const u32x2
								  *)(k_lds +
								     row * RB +
								     piece * 16 +
								     (quarter &
								      1) *
									     8));
					}
#pragma unroll
					for (int n = 0; n < NC; n++)
						score[n][h] = mma16<T>(
							w, q[n][d],
							score[n][h]);
				}
			}
			wait_lds();
			if (more) {
				copy4_to_lds(entry(t + 2 * W),
					     lds_at(entries[wave][turn ^ 1]));
				request(c.k_cache, c.k_page, c.k_slot,
					c.k_head, t + W, pages1, whole1, false,
					k_at);
			}

			/* Weights, in two parts of T: the matrix units have
			 * the time.  Rounded to one, as those of chunks are,
			 * they would move results by as much as the results'
			 * own rounding (together 2.3e-3 of their size in
			 * bfloat16 and 2.9e-4 in float16, where this leaves
			 * 1.7e-3 and 2.1e-4), for 11.4 us instead of 11.7 (a
			 * token over 611 keys), 95.0 instead of 95.6 (over
			 * 120001), 20.8 instead of 21.7 (drafts of 6). */
			const bool masked = valid != ~0ull ||
					    key0 + TILE - 1 > all ||
					    key0 < any_low;
			u32x4 weight[NC][SUBS], rest[NC][SUBS];
#pragma unroll
			for (int n = 0; n < NC; n++) {
				float x[8 * SUBS];

#pragma unroll
				for (int h = 0; h < 2 * SUBS; h++)
#pragma unroll
					for (int j = 0; j < 4; j++)
						x[4 * h + j] = score[n][h][j];
				if (masked) {
					rarely();
					/* As seen from the first key. */
					const uint64_t shown =
						valid >> 4 * quarter;
					const int to = lim[n] - key0 -
						       4 * quarter;
					const int after = low[n] - key0 -
							  4 * quarter;
#pragma unroll
					for (int e = 0; e < 8 * SUBS; e++) {
						const int j = 16 * (e >> 2) +
							      (e & 3);
						const bool sees =
							(shown >> j & 1) &
							(j <= to) & (j > after);

						x[e] = sees ? x[e] : -INFINITY;
					}
				}
				float most = x[0];
#pragma unroll
				for (int e = 1; e < 8 * SUBS; e++)
					most = fmaxf(most, x[e]);
				f32x2 y = odd_even_quarters(most);
				y = halves(fmaxf(y[0], y[1]));
				most = fmaxf(y[0], y[1]);
				if (__any(sm[n].behind(most, f.c))) {
					const float keep =
						sm[n].follow(most, f.c);
#pragma unroll
					for (int d = 0; d < D / 16; d++)
						out[n][d] *= keep;
				}
				const float unit = sm[n].unit(f.c);
#pragma unroll
				for (int e = 0; e < 8 * SUBS; e++) {
					x[e] = __builtin_amdgcn_exp2f(
						__builtin_fmaf(x[e], f.c,
							       -unit));
					sm[n].sum += x[e];
				}
#pragma unroll
				for (int e = 0; e < 4 * SUBS; e++) {
					const u32x2 w = split2<T>(x[2 * e],
								  x[2 * e + 1]);

					weight[n][e / 4][e % 4] = w[0];
					rest[n][e / 4][e % 4] = w[1];
				}
			}

			/* Values: O^T += V^T P^T. */
			if (more)
				wait_loads<NI + 1>();
			else
				wait_loads<0>();
			auto value = [&](int sub, int d) {
				if constexpr (sizeof(C) == 2) {
					const int row = 32 * sub +
							4 * quarter +
							(col >> 2);
					const int piece =
						(2 * d + ((col & 3) >> 1)) ^
						N::turn_v(row);
					const char *at = v_lds + row * RB +
							 piece * 16 +
							 (col & 1) * 8;
					const u32x2 lo = read_keys4(at);
					const u32x2 hi =
						read_keys4(at + 16 * RB);

					return u32x4{ lo[0], lo[1], hi[0],
						      hi[1] };
				} else {
					const int n = col >> 1;
					const int row =
						32 * sub + (n < 4 ? 0 : 12) +
						4 * quarter + n;
					const int piece = d ^ N::turn_v(row);

					return widen8<T>(read_keys8(
						v_lds + row * RB +
						piece * 16 + (col & 1) * 8));
				}
			};
			/* The 4 values of key j that go into out[.][d]. */
			auto four = [&](int j, int d, float *x) {
				const int byte = (16 * d + 4 * quarter) *
						 (int)sizeof(C);
				const char *at =
					v_lds + j * RB +
					((byte >> 4) ^ N::turn_v(j)) * 16 +
					(byte & 15);

				if constexpr (sizeof(C) == 2) {
					const u32x2 w = *(const u32x2 *)at;
					const T *v = (const T *)&w;
#pragma unroll
					for (int e = 0; e < 4; e++)
						x[e] = (float)v[e];
				} else {
					const unsigned w =
						*(const unsigned *)at;
					const f32x2 lo =
						__builtin_amdgcn_cvt_pk_f32_fp8(
							w, false);
					const f32x2 hi =
						__builtin_amdgcn_cvt_pk_f32_fp8(
							w, true);

					x[0] = lo[0];
					x[1] = lo[1];
					x[2] = hi[0];
					x[3] = hi[1];
				}
			};
			/* 0 * inf is no number.  Where some rows see a key and
			 * others do not, and its values are not all finite,
			 * the rows that see it get these added one by one,
			 * and the product takes zeros in their place. */
			bool odd = false;

			if (masked && !alike)
#pragma unroll 2
				for (int i = 0; i < NI; i++) {
					const u32x4 w =
						*(const u32x4 *)(v_lds +
								 i * 1024 +
								 lane * 16);

					odd |= not_finite<C>(w[0]) |
					       not_finite<C>(w[1]) |
					       not_finite<C>(w[2]) |
					       not_finite<C>(w[3]);
				}
			if (__any(odd)) {
#pragma unroll 1
				for (int j = 0; j < TILE; j++) {
					const int key = key0 + j;
					bool sees[NC];

#pragma unroll
					for (int n = 0; n < NC; n++)
						sees[n] = (valid >> j & 1) &&
							  key <= lim[n] &&
							  key > low[n];
#pragma unroll
					for (int d = 0; d < D / 16; d++) {
						float x[4];

						asm volatile("" ::: "memory");
						four(j, d, x);
#pragma unroll
						for (int n = 0; n < NC; n++)
#pragma unroll
							for (int e = 0; e < 4;
							     e++)
								out[n][d][e] +=
									sees[n] ?
										odd_only(
											x[e]) :
										0.f;
					}
				}
#pragma unroll 1
				for (int i = 0; i < NI; i++) {
					u32x4 *at = (u32x4 *)(v_lds + i * 1024 +
							      lane * 16);
					u32x4 w = *at;

#pragma unroll
					for (int e = 0; e < 4; e++)
						w[e] = finite_only<C>(w[e]);
					*at = w;
				}
				asm volatile("" ::: "memory");
			}
#pragma unroll
			for (int sub = 0; sub < SUBS; sub++)
#pragma unroll
				for (int d = 0; d < D / 16; d++) {
					const u32x4 w = value(sub, d);
#pragma unroll
					for (int n = 0; n < NC; n++) {
						out[n][d] = mma16<T>(
							w, weight[n][sub],
							out[n][d]);
						out[n][d] = mma16<T>(
							w, rest[n][sub],
							out[n][d]);
					}
				}
			wait_lds();
			if (more)
				request(c.v_cache, c.v_page, c.v_slot,
					c.v_head, t + W, pages1, whole1, true,
					v_at);
			pages = pages1;
			whole = whole1;
		}

		/* Join the waves. */
		float *const merge = (float *)lds;
		const float lift = types<T>::lift;

		__syncthreads(); /* all have read their tiles */
#pragma unroll
		for (int n = 0; n < NC; n++) {
			f32x2 y = odd_even_quarters(sm[n].sum);
			y = halves(y[0] + y[1]);
			if (quarter == 0) {
				tops[wave][16 * n + col] = sm[n].top;
				sums[wave][16 * n + col] = y[0] + y[1];
			}
#pragma unroll
			for (int d = 0; d < D / 16; d++)
				*(f32x4 *)(merge +
					   (wave * 16 * NC + 16 * n + col) *
						   N::OUT_ROW +
					   16 * d + 4 * quarter) = out[n][d];
		}
		__syncthreads();
		for (int at = threadIdx.x; at < 16 * NC * (D / 8);
		     at += 64 * W) {
			const int r = at / (D / 8), d = at % (D / 8) * 8;
			const int i = (r0 + r) / group;
			const int head = kh * group + (r0 + r) % group;
			float top = -INFINITY, sum = 0.f, x[8] = {};

			if (r0 + r >= rows)
				continue;
#pragma unroll
			for (int w = 0; w < W; w++)
				top = fmaxf(top, tops[w][r]);
#pragma unroll
			for (int w = 0; w < W; w++) {
				const float *src =
					merge +
					(w * 16 * NC + r) * N::OUT_ROW + d;
				const float m =
					tops[w][r] == -INFINITY ?
						0.f :
						__builtin_amdgcn_exp2f(
							(tops[w][r] - top) *
							f.c);

				sum += m * sums[w][r];
#pragma unroll
				for (int e = 0; e < 8; e++)
					x[e] += m * src[e];
			}
			const int64_t row = s.first + i;
			const float unit = top == -INFINITY ? -INFINITY :
							      top * f.c - lift;

			if (slot >= 0) {
				const int64_t at_row =
					part_at(p, kh, block, slot) + r;
				f32x4 *o = (f32x4 *)(p.narrow_out +
						     at_row * D + d);

				o[0] = f32x4{ x[0], x[1], x[2], x[3] };
				o[1] = f32x4{ x[4], x[5], x[6], x[7] };
				if (d == 0)
					p.narrow_sum[at_row] = f32x2{ unit, sum };
				continue;
			}
			const float inv = sum == 0.f ? 0.f : vs / sum;
			u32x4 o;

#pragma unroll
			for (int e = 0; e < 4; e++)
				o[e] = pack2<T>(x[2 * e] * inv,
						x[2 * e + 1] * inv);
			*(u32x4 *)((T *)a.out + row * a.out_row +
				   head * a.out_head + d) = o;
			if (a.lse && d == 0)
				a.lse[row * c.heads + head] =
					sum == 0.f ?
						-INFINITY :
						(unit +
						 __builtin_amdgcn_logf(sum)) *
							0.693147181f;
		}
		__syncthreads(); /* before the next piece's tiles */
	}
}

template <typename T, typename C, int D>
void launch(const nvs_kv &c, const nvs_kv_attend_args &a, const nvs_plan &p,
	    hipStream_t s)
{
	/* Wide rows of 16 bits: half the waves, as their tiles are twice as
	 * large. */
	constexpr int W = nvs_narrow_waves(D, sizeof(C));
	const dim3 grid(p.narrow_blocks * c.kv_heads);

	if (p.span == 16)
		hipLaunchKernelGGL((narrow_kernel<T, C, D, 1, W>), grid,
				   dim3(64 * W), 0, s, c, a, p);
	else
		hipLaunchKernelGGL((narrow_kernel<T, C, D, 2, W>), grid,
				   dim3(64 * W), 0, s, c, a, p);
}

} /* namespace */

template <typename T, typename C>
hipError_t nvs_narrow(const nvs_kv &c, const nvs_kv_attend_args &a,
		      const nvs_plan &p, hipStream_t s)
{
	if (c.dim == 64)
		launch<T, C, 64>(c, a, p, s);
	else if (c.dim == 128)
		launch<T, C, 128>(c, a, p, s);
	else
		launch<T, C, 256>(c, a, p, s);
	return hipGetLastError();
}

#define INSTANCE(T, C)                                                     \
	template hipError_t nvs_narrow<T, C>(const nvs_kv &,               \
					     const nvs_kv_attend_args &,   \
					     const nvs_plan &,             \
					     hipStream_t);
INSTANCE(bf16_t, bf16_t)
INSTANCE(bf16_t, e4m3_t)
INSTANCE(fp16_t, fp16_t)
INSTANCE(fp16_t, e4m3_t)
