// Attention of one new token per sequence over its pages.
//
//   o = sum_j 2^(x_j - m) v_j / sum_j 2^(x_j - m),   x_j = scale log2(e) q . k_j,   m the running maximum
//
// One pass over k and v, which is what bounds it: 4 head_dim bytes per key and kv head against 8 head_dim flops per query head.
// All tiles (64 keys of one sequence and kv head) of the batch form one list that is cut into stretches of equal cost, one per SM, so
// sequences of any mix of lengths keep all SMs equally busy; a (sequence, kv head) that falls into several stretches is joined by
// the CTA that finishes it last, in the order of the keys (the result does not depend on who that is).
//
// A producer warp follows the page table (32 entries at a time) and feeds a ring of TMA tiles; two groups of four warps take turns
// with the tiles, 16 keys per warp.  The heads of a group share the keys: m16n8k16 takes 16 rows, of which rows 0-7 are the high
// 16-bit parts of up to eight query heads and rows 8-15 the low parts, so f32 accuracy costs no further product, and high and
// low sums of one head meet in the same thread.  The weights go the same way.  mma.sync accumulates only one step of 16 keys; the
// running sums are f32 FMAs, because the tensor cores truncate.  (bf16 parts hold 8 bits each: a third one takes a product of its
// own, in rows 0-7.)
//
// Every wait is bounded; one that runs out is recorded for the host.  A warp whose wait ran out goes on without waiting, so that what
// other CTAs count on is counted, but arrives nowhere in its own any more: a slot is never filled while a copy into it is in flight.
//
// The warps work ahead of one another over the (sequence, kv head) pieces of a stretch: the producer fetches the next piece's
// queries and tiles, the compute warps leave a piece's eight partial results in one of two buffers and go on, and two finishing
// warps join them with what other CTAs and the shared prefix contribute.
//
// B200, f16, 32 heads of 128 on 8: 48 sequences of up to 16001 tokens 259 us (1.66 GB: 6.4 TB/s, 98 % of the copy rate), one of
// 1000 tokens 9.9 us, of which 3 us are the list, lengths and table looked up one after the other.
#include <algorithm>

#include "attention.h"

namespace nhb {

	namespace {

		constexpr int KT		= 64;// keys of a tile
		constexpr int WARPS		= 8;// compute warps, two groups of four
		constexpr int FINISH	= 2;// finishing warps (twelve warps in all leave a thread 168 registers, thirteen 128)
		constexpr int THREADS	= (WARPS + 1 + FINISH) * 32;
		constexpr int MAX_LIST	= 1024;// list entries of a launch
		// What beginning and ending a (sequence, kv head) costs, in tiles: with 0, CTAs that got many short sequences took twice the
		// others' time (64 sequences of up to 700 tokens: 84 us)
		constexpr int UNIT_COST = 2;
		constexpr int ROWS		= 8;// query heads taken together

		__host__ __device__ constexpr int stage_bytes(int d) {
			return 2 * KT * d * 2;
		}
		// Even: the teams take turns with the tiles, so each slot of the ring belongs to one team.  (With an odd depth a slot changes
		// hands, and a team that is done with its own tiles could wait for a slot's next phase before the other team's tile has landed
		// in it: a parity wait that is a phase early passes at once.)
		__host__ __device__ constexpr int n_stages(int d) {
			return d == 128 ? 4 : 8;
		}

		struct decode_head {
			uint64_t full[8];
			uint64_t empty[8];
			uint64_t q_full[2], q_empty[2];// a piece's queries
			uint64_t part_full[2], part_empty[2];// a piece's partial results
			int flag;
			long long scan[THREADS / 32];
		};
		struct part_ml {// per warp and head
			float m[WARPS][ROWS];
			float l[WARPS][ROWS];
		};
		__host__ __device__ constexpr int part_bytes(int d) {
			return WARPS * ROWS * d * 4;
		}
		__host__ __device__ constexpr int smem_bytes(int d) {
			return 1024 + n_stages(d) * stage_bytes(d) + 2 * part_bytes(d) + 2 * ROWS * d * 4 + 2 * static_cast<int>(sizeof(part_ml)) + (MAX_LIST + 1) * 8 +
				MAX_LIST * 8 + static_cast<int>(sizeof(decode_head)) + 64;
		}
		// a slot of the workspace: outputs [8][d], then m[8], l[8]
		__host__ __device__ constexpr int slot_floats(int d) {
			return ROWS * d + 2 * ROWS;
		}

		struct decode_params {
			kv_view c;
			attn_args a;
			attn_prefix pre;
			int row0;// of this launch's first list entry among the rows of `pre`
			int blocks;// groups of eight heads on a kv head
			int skip_pages;// whole pages that the prefix has covered
			int check_pages;// whole pages that all entries say they share
			const int* list;// the whole list (a launch may hold a part of it)
			int list_n;
			float* slots;
			unsigned* counters;
		};

		__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
			asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
		}
		__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
			asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
		}
		template<bool BF16> __device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
			if constexpr (BF16)
				asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
							 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
							 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
			else
				asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
							 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
							 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
		}
		__device__ __forceinline__ void finish_barrier() {
			asm volatile("bar.sync 1, %0;" ::"n"(FINISH * 32) : "memory");
		}

		// (a, b) as high and low parts, bf16 with a third: 8 + 8 + 8 bits
		template<bool BF16> __device__ __forceinline__ void split_row(float a, float b, uint32_t (&r)[3]) {
			split2<BF16>(a, b, r[0], r[1]);
			if constexpr (BF16) {
				const __nv_bfloat162 h = *reinterpret_cast<const __nv_bfloat162*>(&r[0]), l = *reinterpret_cast<const __nv_bfloat162*>(&r[1]);
				const __nv_bfloat162 t = __floats2bfloat162_rn((a - __low2float(h)) - __low2float(l), (b - __high2float(h)) - __high2float(l));
				r[2]				   = *reinterpret_cast<const uint32_t*>(&t);
			}
		}

		// keys of list entry i behind the shared pages; -1: nothing to do for it (padding, or reported as unsound)
		__device__ __forceinline__ int keys_of(const decode_params& p, int i, bool tell) {
			const int s = p.a.seqs[i];
			if (s == -1)
				return -1;
			if (s >= 0 && s < p.c.max_seqs) {
				const int len = p.c.lens[s];
				if (len >= 0 && len <= kv_capacity(p.c) && len >> p.c.page_shift >= p.check_pages)
					return len - (p.skip_pages << p.c.page_shift);
			}
			if (tell)
				atomicCAS(p.c.status, DEV_OK, DEV_KV_BAD);
			return -1;
		}

		// The list in units of cost: every unit -- a list entry's kv head and block of heads -- has UNIT_COST positions and then one per
		// tile; entries without keys have none.  A piece is what a stretch [x, x1) holds of a unit's tiles.
		struct piece_t {
			int i, unit;// list entry, unit of the entry
			int t0, t1;// tiles
			long long first, last;// positions of the unit's first and last tile
		};
		__device__ __forceinline__ bool next_piece(const long long* cum, int n, int units, long long& x, long long x1, piece_t& r) {
			while (x < x1) {
				int lo = 0, hi = n - 1;// the entry with cum[i] * units <= x < cum[i + 1] * units
				while (lo < hi) {
					const int mid = (lo + hi + 1) >> 1;
					if (cum[mid] * units <= x)
						lo = mid;
					else
						hi = mid - 1;
				}
				const long long size = cum[lo + 1] - cum[lo], rest = x - cum[lo] * units;
				r.i				= lo;
				r.unit			= static_cast<int>(rest / size);
				const long long u0 = x - (rest - r.unit * size);
				const long long e  = min(x1, u0 + size);
				r.t0	= static_cast<int>(max(x - u0 - UNIT_COST, 0ll));
				r.t1	= static_cast<int>(max(e - u0 - UNIT_COST, 0ll));
				r.first = u0 + UNIT_COST;
				r.last	= u0 + size - 1;
				x		= e;
				if (r.t1 > r.t0)
					return true;
			}
			return false;
		}

		// One thread's share of a unit's result: head h, V columns from d on, as (maximum, sum, unnormalised outputs)
		template<int V> struct share {
			float m = -INFINITY, l = 0.f;
			float o[V] = {};
			__device__ __forceinline__ void add(float m2, float l2, const float (&o2)[V]) {
				const float top = fmaxf(m, m2), mm = top == -INFINITY ? 0.f : top;
				const float a = ex2(m - mm), b = ex2(m2 - mm);
				m = top;
				l = l * a + l2 * b;
#pragma unroll
				for (int i = 0; i < V; ++i)
					o[i] = o[i] * a + o2[i] * b;
			}
			// n further parts: their maxima and sums ml_step apart, their outputs o_step apart; FLY in flight
			__device__ __forceinline__ void add_parts(const float* pm, const float* pl, long long ml_step, const float* po, long long o_step, int n) {
				constexpr int FLY = 4;
				for (int s0 = 0; s0 < n; s0 += FLY) {
					float m2[FLY], l2[FLY], o2[FLY][V];
#pragma unroll
					for (int j = 0; j < FLY; ++j) {
						const long long s = min(s0 + j, n - 1);
						m2[j]			  = __ldcg(pm + s * ml_step);
						l2[j]			  = __ldcg(pl + s * ml_step);
#pragma unroll
						for (int i = 0; i < V; i += 4) {
							const float4 x = __ldcg(reinterpret_cast<const float4*>(po + s * o_step + i));
							o2[j][i]	   = x.x;
							o2[j][i + 1]   = x.y;
							o2[j][i + 2]   = x.z;
							o2[j][i + 3]   = x.w;
						}
					}
#pragma unroll
					for (int j = 0; j < FLY; ++j)
						if (s0 + j < n)
							add(m2[j], l2[j], o2[j]);
				}
			}
			__device__ __forceinline__ void store(float* out, bool any) const {
				const float inv = any ? 1.f / l : 0.f;
#pragma unroll
				for (int i = 0; i < V; i += 4)
					*reinterpret_cast<float4*>(out + i) = make_float4(o[i] * inv, o[i + 1] * inv, o[i + 2] * inv, o[i + 3] * inv);
			}
		};

		template<int D, bool BF16> __global__ void __launch_bounds__(THREADS, 1)
			attn_decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ decode_params p) {
			static_assert(n_stages(D) % 2 == 0, "a slot belongs to one team");
			constexpr int PANELS = D / 64, NST = n_stages(D), STAGE = stage_bytes(D), PANEL = KT * 128;
			extern __shared__ unsigned char smem_raw[];
			unsigned char* base	 = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
			float* mo			 = reinterpret_cast<float*>(base + NST * STAGE);// [2][WARPS][ROWS][D]
			float* qs			 = mo + 2 * WARPS * ROWS * D;// [2][ROWS][D]
			part_ml* ms			 = reinterpret_cast<part_ml*>(qs + 2 * ROWS * D);// [2]
			long long* cum		 = reinterpret_cast<long long*>(ms + 2);// [n + 1] cost of a unit, summed over the list
			int2* entry			 = reinterpret_cast<int2*>(cum + MAX_LIST + 1);// [n] sequence, keys of its own (behind the shared ones)
			decode_head* hd		 = reinterpret_cast<decode_head*>(entry + MAX_LIST);
			const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
			const int n = p.a.n, units = p.c.kv_heads * p.blocks;
			if (tid == 0) {
				for (int s = 0; s < NST; ++s) {
					mbar_init(&hd->full[s], 1);
					mbar_init(&hd->empty[s], 4);
				}
				for (int b = 0; b < 2; ++b) {
					mbar_init(&hd->q_full[b], 1);
					mbar_init(&hd->q_empty[b], WARPS);
					mbar_init(&hd->part_full[b], WARPS);
					mbar_init(&hd->part_empty[b], FINISH);
				}
				fence_mbar_init();
				cum[0] = 0;
			}
			pdl_launch_dependents();
			pdl_wait_prior_grids();
			__syncthreads();
			// ---- the list: running sums of each entry's cost ----
			long long before = 0;
			for (int i0 = 0; i0 < n; i0 += THREADS) {
				const int i	 = i0 + tid;
				const int kk = i < n ? keys_of(p, i, blockIdx.x == 0) : -1;
				if (i < n)
					entry[i] = make_int2(p.a.seqs[i], kk);
				long long x = kk > 0 ? (kk + KT - 1) / KT + UNIT_COST : 0;
#pragma unroll
				for (int o = 1; o < 32; o <<= 1) {
					const long long y = __shfl_up_sync(0xffffffffu, x, o);
					if (lane >= o)
						x += y;
				}
				if (lane == 31)
					hd->scan[warp] = x;
				__syncthreads();
				long long sum = before;
				for (int w = 0; w < warp; ++w)
					sum += hd->scan[w];
				if (i < n)
					cum[i + 1] = sum + x;
				for (int w = warp; w < THREADS / 32; ++w)
					sum += hd->scan[w];
				before = sum;
				__syncthreads();
			}
			const long long total = before * units;
			// CTAs with a stretch: of at least two tiles, which its two teams take side by side in the time of one -- half the parts to join
			const int parts		  = static_cast<int>(min((total + 1) / 2, static_cast<long long>(gridDim.x)));
			const long long x0	  = static_cast<int>(blockIdx.x) < parts ? blockIdx.x * total / parts : 0;
			const long long x1	  = static_cast<int>(blockIdx.x) < parts ? (blockIdx.x + 1) * total / parts : 0;

			if (warp == WARPS) {
				// ---------------- producer ----------------
				const int box_rows = p.c.page_tokens < 64 ? p.c.page_tokens : 64;
				int s			   = 0;
				uint32_t ph		   = 1;
				bool ok			   = true;
				int number = 0;// of the piece
				int issued = 0, q_issued = 0;// copies of tiles and of queries (lane 0)
				long long x = x0;
				piece_t at, then;
				bool more = next_piece(cum, n, units, x, x1, at);
				// 32 page numbers from a piece's first on, one per lane: those of the next piece are on their way while this one's tiles are
				// issued.  A number that is none is reported where it is used, and read as page 0.
				const auto pages_from = [&](const piece_t& a, int j) {
					const int2 e	= entry[a.i];
					const int pages = p.skip_pages + kv_pages_of(p.c, e.y);
					return j + lane < pages ? p.c.table[static_cast<size_t>(e.x) * p.c.max_pages + j + lane] : 0;
				};
				const auto first_page = [&](const piece_t& a) {
					return p.skip_pages + ((a.t0 * KT) >> p.c.page_shift);
				};
				const auto sound = [&](int page) {
					if (page >= 0 && page < p.c.n_pages)
						return page;
					atomicCAS(p.c.status, DEV_OK, DEV_KV_BAD);
					return 0;
				};
				int ahead = more ? pages_from(at, first_page(at)) : 0;
				for (; more && ok; ++number) {
					const int kvh  = at.unit / p.blocks;
					const int keys = entry[at.i].y;
					if (lane == 0) {
						const int head0 = (at.unit - kvh * p.blocks) * ROWS, b = number & 1;
						const int bytes = min(ROWS, p.a.group - head0) * D * 4;
						if (!mbar_wait(&hd->q_empty[b], ((number >> 1) & 1) ^ 1)) {
							ok = false;
						} else {
							mbar_expect_tx(&hd->q_full[b], bytes);
							++q_issued;
							bulk_g2s_plain(smem_u32(qs + b * ROWS * D), p.a.q + static_cast<long long>(at.i) * p.a.ldq + static_cast<long long>(kvh * p.a.group + head0) * D, bytes, &hd->q_full[b]);
						}
					}
					ok		  = __shfl_sync(0xffffffffu, ok, 0);
					int page0 = first_page(at), page = sound(ahead);
					more = next_piece(cum, n, units, x, x1, then);
					ahead = more ? pages_from(then, first_page(then)) : 0;
					for (int t = at.t0; t < at.t1 && ok; ++t) {
						const int key0	= t * KT;// behind the shared pages
						const int boxes = (min(KT, keys - key0) + box_rows - 1) / box_rows;
						const int j0	= p.skip_pages + (key0 >> p.c.page_shift);
						if (j0 + ((boxes * box_rows - 1) >> p.c.page_shift) >= page0 + 32) {
							page0 = j0;
							page  = sound(pages_from(at, j0));
						}
						if (lane == 0) {
							if (!mbar_wait(&hd->empty[s], ph)) {
								ok = false;
							} else {
								mbar_expect_tx(&hd->full[s], boxes * 2 * PANELS * box_rows * 128);
								++issued;
							}
						}
						ok = __shfl_sync(0xffffffffu, ok, 0);
						// a lane per copy: box, panel of head_dim, k or v (one lane issuing all of a tile's 4 to 16 took longer than the copies)
						const int box = lane / (2 * PANELS), panel = lane % (2 * PANELS);
						const int k	  = key0 + box * box_rows;
						const int pg  = __shfl_sync(0xffffffffu, page, (p.skip_pages + (k >> p.c.page_shift) - page0) & 31);
						if (box < boxes && ok)
							tma_load_2d(smem_u32(base) + s * STAGE + panel * PANEL + box * box_rows * 128, panel < PANELS ? &map_k : &map_v, (panel % PANELS) * 64,
								((pg * p.c.kv_heads + kvh) << p.c.page_shift) + (k & (p.c.page_tokens - 1)), &hd->full[s]);
						__syncwarp();
						if (++s == NST) {
							s = 0;
							ph ^= 1;
						}
					}
					at = then;
				}
				// the last copy into each buffer has landed before the block ends
				if (lane == 0) {
					for (int i = max(0, issued - NST); i < issued; ++i)
						ok = mbar_wait(&hd->full[i % NST], (i / NST) & 1) && ok;
					for (int i = max(0, q_issued - 2); i < q_issued; ++i)
						ok = mbar_wait(&hd->q_full[i & 1], (i >> 1) & 1) && ok;
					if (!ok)
						atomicExch(p.c.status, DEV_TIMEOUT_EMPTY);
				}
				return;
			}

			if (warp > WARPS) {
				// ---------------- finish ----------------
				constexpr int PER = FINISH * 32 / ROWS, V = D / PER;// threads of a head, columns of a thread
				const int ft = tid - (WARPS + 1) * 32, h = ft / PER, d = (ft % PER) * V;
				bool ok = true;
				if (p.check_pages > 0) {
					// entries whose claim to the shared pages does not hold: compared with the first entry that is not padding
					int first = -1;
					for (int i = lane; first < 0 && i - lane < p.list_n; i += 32) {
						const int seq	 = i < p.list_n ? p.list[i] : -1;
						const unsigned b = __ballot_sync(0xffffffffu, seq != -1);
						if (b)
							first = __shfl_sync(0xffffffffu, seq, __ffs(b) - 1);
					}
					if (first >= 0 && first < p.c.max_seqs) {// an unsound one has been reported where it stands
						const int* ref = p.c.table + static_cast<size_t>(first) * p.c.max_pages;
						bool same	   = true;
						const long long all = static_cast<long long>(n) * p.check_pages;
#pragma unroll 4
						for (long long y = blockIdx.x * (FINISH * 32ll) + ft; y < all; y += gridDim.x * (FINISH * 32ll)) {
							const int i = static_cast<int>(y / p.check_pages), j = static_cast<int>(y - static_cast<long long>(i) * p.check_pages);
							if (entry[i].y >= 0)
								same = same && p.c.table[static_cast<size_t>(entry[i].x) * p.c.max_pages + j] == ref[j];
						}
						if (!same)
							atomicCAS(p.c.status, DEV_OK, DEV_KV_BAD);
					}
				}
				// the part of the keys that the batch shares
				const auto add_prefix = [&](share<V>& r, int i, int kvh, int head) {
					const long long row = kvh * p.pre.stride + static_cast<long long>(p.row0 + i) * p.a.group + head;
					const float* ml		= reinterpret_cast<const float*>(p.pre.ml + row);
					r.add_parts(ml, ml + 1, 0, p.pre.o + row * D + d, 0, p.pre.any);
				};
				piece_t at;
				long long x = x0;
				for (int number = 0; next_piece(cum, n, units, x, x1, at); ++number) {
					const int kvh = at.unit / p.blocks, head0 = (at.unit - kvh * p.blocks) * ROWS;
					const bool mine = h < min(ROWS, p.a.group - head0);
					const int b		= number & 1;
					// who holds the unit's first and last tile: stretch k begins at k * total / parts
					const long long unit = static_cast<long long>(at.i) * units + at.unit;
					const int c0 = static_cast<int>(((at.first + 1) * parts - 1) / total), c1 = static_cast<int>(((at.last + 1) * parts - 1) / total);
					float* out	 = p.a.out + static_cast<long long>(at.i) * p.a.ldo + static_cast<long long>(kvh * p.a.group + head0 + h) * D + d;
					share<V> r;
					if (c0 == c1 && mine)
						add_prefix(r, at.i, kvh, head0 + h);// while the keys are still being read
					if (ok && !mbar_wait(&hd->part_full[b], (number >> 1) & 1)) {
						ok = false;
						atomicExch(p.c.status, DEV_TIMEOUT_DRAIN);
					}
					const part_ml& pm = ms[b];
					float top		  = -INFINITY;
#pragma unroll
					for (int w = 0; w < WARPS; ++w)
						top = fmaxf(top, pm.m[w][h]);
					const float mm = top == -INFINITY ? 0.f : top;
					float sum	   = 0.f;
					float v[V]	   = {};
#pragma unroll
					for (int w = 0; w < WARPS; ++w) {
						const float f = ex2(pm.m[w][h] - mm);
						sum			  = fmaf(pm.l[w][h], f, sum);
#pragma unroll
						for (int i = 0; i < V; i += 4) {
							const float4 y = *reinterpret_cast<const float4*>(mo + ((b * WARPS + w) * ROWS + h) * D + d + i);
							v[i]		   = fmaf(y.x, f, v[i]);
							v[i + 1]	   = fmaf(y.y, f, v[i + 1]);
							v[i + 2]	   = fmaf(y.z, f, v[i + 2]);
							v[i + 3]	   = fmaf(y.w, f, v[i + 3]);
						}
					}
					__syncwarp();
					if (lane == 0 && ok)
						mbar_arrive(&hd->part_empty[b]);
					if (c0 == c1) {
						if (mine) {
							r.add(top, sum, v);
							r.store(out, true);
						}
					} else {
						float* slot = p.slots + (blockIdx.x + unit) * slot_floats(D);// distinct: along the list, block or unit moves on
						if (mine) {
#pragma unroll
							for (int i = 0; i < V; i += 4)
								__stcg(reinterpret_cast<float4*>(slot + h * D + d + i), make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]));
							if (d == 0) {
								__stcg(slot + ROWS * D + h, top);
								__stcg(slot + ROWS * D + ROWS + h, sum);
							}
						}
						__threadfence();
						finish_barrier();
						if (ft == 0) {
							const bool last = atomicAdd(p.counters + unit, 1u) == static_cast<unsigned>(c1 - c0);
							if (last)
								p.counters[unit] = 0u;// ready for the next launch
							__threadfence();
							hd->flag = last;
						}
						finish_barrier();
						const bool last = *reinterpret_cast<volatile int*>(&hd->flag) != 0;
						if (last && mine) {
							const float* first = p.slots + (c0 + unit) * slot_floats(D);
							add_prefix(r, at.i, kvh, head0 + h);
							r.add_parts(first + ROWS * D + h, first + ROWS * D + ROWS + h, slot_floats(D), first + h * D + d, slot_floats(D), c1 - c0 + 1);
							r.store(out, true);
						}
						finish_barrier();// the flag is read
					}
				}
				// ---- entries without keys of their own: the shared part alone, or zeros ----
				for (int i = blockIdx.x; i < n; i += gridDim.x) {
					if (entry[i].y != 0)
						continue;
					for (int u = 0; u < units; ++u) {
						const int kvh = u / p.blocks, head0 = (u - kvh * p.blocks) * ROWS;
						if (h < min(ROWS, p.a.group - head0)) {
							share<V> r;
							add_prefix(r, i, kvh, head0 + h);
							r.store(p.a.out + static_cast<long long>(i) * p.a.ldo + static_cast<long long>(kvh * p.a.group + head0 + h) * D + d, p.pre.any != 0);
						}
					}
				}
				return;
			}

			// ---------------- compute ----------------
			const int g = lane >> 2, t4 = lane & 3;// fragment row (head) and column pair
			const int team = warp >> 2, wk = (warp & 3) * 16;// this warp's 16 keys of its team's tiles
			bool ok	  = true;
			int count = 0;// tiles of this CTA so far
			piece_t at;
			long long x = x0;
			for (int number = 0; next_piece(cum, n, units, x, x1, at); ++number) {
				const int kvh = at.unit / p.blocks, head0 = (at.unit - kvh * p.blocks) * ROWS;
				const int heads = min(ROWS, p.a.group - head0);
				const int keys	= entry[at.i].y;
				// ---- this thread's part of the queries: head g, columns 16 j + 2 t4 + {0, 1, 8, 9} ----
				uint32_t qa[D / 16][4], q3[BF16 ? D / 16 : 1][2];
				float factor = 0.f;// scores back to their size, in powers of two
				{
					const int b = number & 1;
					if (ok && !mbar_wait(&hd->q_full[b], (number >> 1) & 1)) {
						ok = false;
						atomicExch(p.c.status, DEV_TIMEOUT_FULL);
					}
					const float* src = qs + (b * ROWS + g) * D + 2 * t4;
					float f = 1.f, back = 1.f;
					if constexpr (!BF16) {
						float amax = 0.f;
#pragma unroll
						for (int j = 0; j < D / 8; ++j) {
							const float2 v = *reinterpret_cast<const float2*>(src + 8 * j);
							amax		   = fmaxf(amax, fmaxf(fabsf(v.x), fabsf(v.y)));
						}
						amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
						amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
						f	 = row_scaling(amax, &back);
					}
					factor = back * p.a.scale2;
#pragma unroll
					for (int j = 0; j < D / 8; ++j) {
						float2 v = *reinterpret_cast<const float2*>(src + 8 * j);
						if (g >= heads)
							v = make_float2(0.f, 0.f);// the buffer holds anything there
						uint32_t a[3];
						split_row<BF16>(v.x * f, v.y * f, a);
						qa[j >> 1][2 * (j & 1)]		= a[0];
						qa[j >> 1][2 * (j & 1) + 1] = a[1];
						if constexpr (BF16)
							q3[j >> 1][j & 1] = a[2];
					}
					if (g >= heads)
						factor = p.a.scale2;
					__syncwarp();
					if (lane == 0 && ok)
						mbar_arrive(&hd->q_empty[b]);
				}
				float m = -INFINITY, l = 0.f;
				float o[D / 8][2];
#pragma unroll
				for (int j = 0; j < D / 8; ++j)
					o[j][0] = o[j][1] = 0.f;
				for (int t = at.t0; t < at.t1; ++t, ++count) {
					if ((count & 1) != team)
						continue;
					const int s = count % NST;
					if (ok && !mbar_wait(&hd->full[s], (count / NST) & 1)) {
						ok = false;
						atomicExch(p.c.status, DEV_TIMEOUT_FULL);
					}
					const uint32_t st = smem_u32(base) + s * STAGE;
					const int left	  = keys - t * KT - wk;// valid keys from this warp's first on
					if (left < 16) {
						// rows past the sequence's end hold anything: their weights are zero, and so must the values be
						for (int r = max(left, 0); r < 16; ++r)
							for (int c = 0; c < PANELS; ++c)
								if (lane < 8)
									*reinterpret_cast<uint4*>(base + s * STAGE + (PANELS + c) * PANEL + (wk + r) * 128 + lane * 16) = make_uint4(0, 0, 0, 0);
						__syncwarp();
					}
					// ---- scores: 8 heads (high and low parts) x 16 keys ----
					float s0[4] = { 0.f, 0.f, 0.f, 0.f }, s1[4] = { 0.f, 0.f, 0.f, 0.f };
					{
						const int r = wk + (lane & 7) + ((lane >> 4) << 3);// matrices 0, 1: keys 0-7, matrices 2, 3: keys 8-15
#pragma unroll
						for (int j = 0; j < D / 16; ++j) {
							uint32_t kb[4];
							const int chunk = ((2 * j) & 7) + ((lane >> 3) & 1);
							ldsm4(st + (j >> 2) * PANEL + r * 128 + ((chunk ^ (r & 7)) << 4), kb);
							mma16816<BF16>(s0, qa[j], kb[0], kb[1]);
							mma16816<BF16>(s1, qa[j], kb[2], kb[3]);
							if constexpr (BF16) {
								const uint32_t a[4] = { q3[j][0], 0u, q3[j][1], 0u };
								mma16816<BF16>(s0, a, kb[0], kb[1]);
								mma16816<BF16>(s1, a, kb[2], kb[3]);
							}
						}
					}
					float x4[4] = { (s0[0] + s0[2]) * factor, (s0[1] + s0[3]) * factor, (s1[0] + s1[2]) * factor, (s1[1] + s1[3]) * factor };
					if (left < 16) {
#pragma unroll
						for (int j = 0; j < 4; ++j)
							if (2 * t4 + (j & 1) + 8 * (j >> 1) >= left)
								x4[j] = -INFINITY;
					}
					float top = fmaxf(fmaxf(x4[0], x4[1]), fmaxf(x4[2], x4[3]));
					top		  = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
					top		  = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
					top		  = fmaxf(top, m);
					const float mm	 = top == -INFINITY ? 0.f : top;
					const float keep = ex2(m - mm);
					m				 = top;
					float w[4];
#pragma unroll
					for (int j = 0; j < 4; ++j)
						w[j] = ex2(x4[j] - mm + WEIGHT_BITS<BF16>);
					l = fmaf(l, keep, (w[0] + w[1]) + (w[2] + w[3]));
					uint32_t p0[3], p1[3];
					split_row<BF16>(w[0], w[1], p0);
					split_row<BF16>(w[2], w[3], p1);
					const uint32_t pa[4] = { p0[0], p0[1], p1[0], p1[1] }, p3[4] = { BF16 ? p0[2] : 0u, 0u, BF16 ? p1[2] : 0u, 0u };
					const int r = wk + (lane & 15);// matrices 0, 2: keys 0-7, matrices 1, 3: keys 8-15
#pragma unroll
					for (int j = 0; j < D / 16; ++j) {
						uint32_t vb[4];
						const int chunk = ((2 * j) & 7) + (lane >> 4);
						ldsm4_t(st + (PANELS + (j >> 2)) * PANEL + r * 128 + ((chunk ^ (r & 7)) << 4), vb);
						float c0[4] = { 0.f, 0.f, 0.f, 0.f }, c1[4] = { 0.f, 0.f, 0.f, 0.f };
						if constexpr (BF16) {
							mma16816<BF16>(c0, p3, vb[0], vb[1]);
							mma16816<BF16>(c1, p3, vb[2], vb[3]);
						}
						mma16816<BF16>(c0, pa, vb[0], vb[1]);
						mma16816<BF16>(c1, pa, vb[2], vb[3]);
						o[2 * j][0]		= fmaf(o[2 * j][0], keep, c0[0] + c0[2]);
						o[2 * j][1]		= fmaf(o[2 * j][1], keep, c0[1] + c0[3]);
						o[2 * j + 1][0] = fmaf(o[2 * j + 1][0], keep, c1[0] + c1[2]);
						o[2 * j + 1][1] = fmaf(o[2 * j + 1][1], keep, c1[1] + c1[3]);
					}
					if (left < 16)
						fence_proxy_async();// the zeroed rows, before the next tile is copied over them
					__syncwarp();
					if (lane == 0 && ok)
						mbar_arrive(&hd->empty[s]);
				}
				// ---- this warp's part of the piece ----
				l += __shfl_xor_sync(0xffffffffu, l, 1);
				l += __shfl_xor_sync(0xffffffffu, l, 2);
				const int b = number & 1;
				if (ok && !mbar_wait(&hd->part_empty[b], ((number >> 1) & 1) ^ 1)) {
					ok = false;
					atomicExch(p.c.status, DEV_TIMEOUT_EMPTY);
				}
				if (t4 == 0) {
					ms[b].m[warp][g] = m;
					ms[b].l[warp][g] = l;
				}
				if (g < heads)
#pragma unroll
					for (int j = 0; j < D / 8; ++j)
						*reinterpret_cast<float2*>(mo + ((b * WARPS + warp) * ROWS + g) * D + 8 * j + 2 * t4) = make_float2(o[j][0], o[j][1]);
				__syncwarp();
				if (lane == 0 && ok)
					mbar_arrive(&hd->part_full[b]);
			}
		}

		int list_per_launch(const kv_view& c, const attn_args& a) {
			const int units = c.kv_heads * ((a.group + ROWS - 1) / ROWS);
			return std::min(MAX_LIST, NHB_KV_COUNTERS / units);
		}

	}

	size_t attn_decode_ws_bytes(const nhb_ctx* ctx, const kv_view& c, const attn_args& a) {
		const size_t units = static_cast<size_t>(c.kv_heads) * ((a.group + ROWS - 1) / ROWS);
		return (ctx->sm_count + std::min<size_t>(a.n, list_per_launch(c, a)) * units) * slot_floats(c.head_dim) * sizeof(float);
	}

	int launch_attn_decode(nhb_ctx* ctx, const kv_view& c, const attn_args& a, const attn_prefix& pre, void* ws) {
		CUtensorMap mk, mv;
		if (!make_page_map(&mk, c, c.k, a.layer) || !make_page_map(&mv, c, c.v, a.layer))
			return fail(ctx, NHB_ERR_CUDA, "nhb_attn_decode: cuTensorMapEncodeTiled failed");
		auto kern = c.head_dim == 128 ? (c.bf16 ? attn_decode_kernel<128, true> : attn_decode_kernel<128, false>)
									  : (c.bf16 ? attn_decode_kernel<64, true> : attn_decode_kernel<64, false>);
		const int smem = smem_bytes(c.head_dim);
		if (int rc = kv_allow_smem(ctx, reinterpret_cast<const void*>(kern), smem); rc != NHB_OK)
			return rc;
		const int most = list_per_launch(c, a);
		for (int i0 = 0; i0 < a.n; i0 += most) {
			decode_params p{};
			p.c			 = c;
			p.a			 = a;
			p.a.n		 = std::min(most, a.n - i0);
			p.a.seqs	 = a.seqs + i0;
			p.a.q		 = a.q + i0 * a.ldq;
			p.a.out		 = a.out + i0 * a.ldo;
			p.pre		 = pre;
			p.row0		 = i0;
			p.blocks	 = (a.group + ROWS - 1) / ROWS;
			p.check_pages = a.shared_pages;
			p.skip_pages  = pre.any ? a.shared_pages : 0;
			p.list		  = a.seqs;
			p.list_n	  = a.n;
			p.slots		 = static_cast<float*>(ws);
			p.counters	 = kv_counters(ctx);
			cudaError_t e = kv_launch(ctx, kern, dim3(ctx->sm_count), dim3(THREADS), smem, mk, mv, p);
			if (e != cudaSuccess)
				return fail_cuda(ctx, e, "attn_decode launch");
		}
		return NHB_OK;
	}

}
