// Attention of many rows over the paged cache on the tensor cores (tcgen05): whole prompts, causal and packed, and the prefix that
// a decode batch shares.
//
//   x_j = scale log2(e) q . k_j,   m' = max(m, x),   l' = l 2^(m - m') + sum 2^(x_j - m'),   o' = o 2^(m - m') + sum 2^(x_j - m') v_j
//
// f32 accuracy from 16-bit products: a query row (f16: scaled by a power of two) enters as PARTS 16-bit parts (f16: two, 2^-22;
// bf16: three, 2^-24), the weights likewise, k and v are 16-bit to begin with.  That is PARTS products where one would do for 16-bit
// rows, and it is what bounds the kernel: 4 head_dim PARTS flops per (row, key).  The tensor cores add into their f32 accumulators by
// truncation, so one accumulator never holds more than a tile of KT keys; the running sums are f32 FMAs in registers.
//
// Rows are (token, query head of the group) pairs, token-major, so that all heads of a group read a tile of k and v once and short
// prompts still fill tiles of 128 rows.  A CTA runs two chains, each S = Q K^T -> softmax -> O = P V, that take turns on the tensor
// cores: while one chain's warps do the softmax, the other chain's products run.  The chains are two row tiles over the same keys
// (TWO: half the k and v traffic) or the even and odd key tiles of one row tile, joined at the end (more CTAs for small calls).
//   warp 0       follows the page table and copies k and v tiles (TMA, 128-byte swizzle) into a ring
//   warp 1       issues the products; P comes from tensor memory, where the softmax warps leave it over S
//   warps 2, 3   watch the ring, and clean v tiles that some row may see only in part: rows past the end become zero, and so do
//                infinities and NaN (0 * inf would reach rows that may not see them; rows that may get them back at the end)
//   warps 4-19   softmax, two threads per row, and the running sums (head_dim / 2 registers each)
// Every wait is bounded; one that runs out is recorded for the host.  A warp whose wait ran out arrives nowhere any more, so that what waits for
// it stops too, and the block ends only after its copies and products.
//
// B200, f16, 32 heads of 128 on 8: 8192 tokens 1017 us (541 TFLOP/s of the formula, 1082 on the tensor cores; 890 in a burst, before the
// power limit brings the clock down), 2048 tokens 94 us, 77 tokens 16 us.  A step (one chain's scores and P V, 32
// m128n128k16) takes 2950 cycles of which the tensor cores need 2070; what is left is a chain's own way round: 2300 cycles of
// softmax beside the other chain's, 1030 of P V, 900 to take the product.  The compiler spills: a warp and step make 10 loads and 3 stores of
// local memory (counted: 1.40 M loads for 16896 steps).
// The grid is row tiles x kv heads and a CTA walks all keys of its rows, so a few rows behind a long context leave most SMs idle: 4 rows behind
// 16000 cached tokens take 256 us where a decode step of that sequence takes 21, and the time grows with the context.
#include <algorithm>

#include "attention.h"

namespace nhb {

	namespace {

		constexpr int PT	   = 640;// threads
		constexpr int TILE	   = 128;// rows of a tile = tensor-memory lanes

		constexpr int parts_of(bool bf16) {
			return bf16 ? 3 : 2;
		}
		constexpr int KT = 128;// keys of a tile
		// Score buffers in tensor memory: 512 columns hold the shared product O (head_dim) and either three buffers of 128 (two parts: the
		// weights lie over the scores) or two and the third parts beside them
		constexpr int score_buffers(bool bf16) {
			return bf16 ? 2 : 3;
		}
		constexpr bool two_fits(int d, bool bf16) {
			return !(bf16 && d == 128);// two row tiles of queries in three parts leave no room for the ring
		}
		constexpr int q_bytes(int d, bool bf16, bool two) {
			return parts_of(bf16) * (two ? 2 : 1) * TILE * d * 2;
		}
		constexpr int slot_bytes(int d) {
			return KT * d * 2;
		}
		constexpr int ring_slots(int d, bool bf16, bool two) {
			const int n = (224 * 1024 - q_bytes(d, bf16, two)) / slot_bytes(d);
			return n > 8 ? 8 : n;
		}

		struct prompt_head {
			uint64_t full[8], empty[8];
			uint64_t s_full[3], p_full[3];// per score buffer
			uint64_t o_full[2];// per chain
			uint64_t q_full;
			uint64_t drain;// all products have run
			union {
				float back[2 * TILE];// before the first tile: what undoes a row's scaling, times scale log2(e)
				float half[2][2][TILE];// per chain and half of the columns: a row's largest score of the tile; at the end its sum
				int scan[PT / 32];// at the start
			};
			uint32_t tmem;
			int odd;// an infinity or NaN was taken out of v
			int entry, total;
			int tile, seq, q_row, count, len;// what the CTA works on
		};
		// The swizzle wants 1024-byte alignment, which the dynamic shared memory of a kernel without static shared memory has; where a
		// block's 227 KB leave no room to make sure, the kernel checks
		constexpr int prompt_smem(int d, bool bf16, bool two) {
			const int n = 1024 + q_bytes(d, bf16, two) + ring_slots(d, bf16, two) * slot_bytes(d) + static_cast<int>(sizeof(prompt_head));
			return n < 227 * 1024 ? n : 227 * 1024;
		}

		struct prompt_params {
			kv_view c;
			attn_args a;
			// prefix (splits > 0): rows are (list entry, head) pairs, the keys those of the first entry's shared pages
			float* o;
			float2* ml;
			int splits, tiles_per_split;
		};

		// ---- tensor-memory access: this warp's 32 lanes, 16 or 8 columns ----
		__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t (&r)[16]) {
			asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
						 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
						 "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
						 : "r"(addr)
						 : "memory");
		}
		// the registers pass through the wait so that no use of them is scheduled ahead of it
		__device__ __forceinline__ void tmem_ld_wait16(uint32_t (&r)[16]) {
			asm volatile("tcgen05.wait::ld.sync.aligned;"
						 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]),
						 "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
						 :
						 : "memory");
		}
		__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t (&r)[8]) {
			asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]),
				"r"(r[7])
				: "memory");
		}
		__device__ __forceinline__ void tmem_st_wait() {
			asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
		}

		// ---- products: A from shared memory (queries) or tensor memory (weights), B from shared memory ----
		__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t add) {
			asm volatile(
				"{\n"
				".reg .pred p;\n"
				".reg .b64 da, db;\n"
				"setp.ne.b32 p, %6, 0;\n"
				"mov.b64 da, {%1, %2};\n"
				"mov.b64 db, {%3, %4};\n"
				"tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n"
				"}\n" ::"r"(d),
				"r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(add)
				: "memory");
		}
		__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t add) {
			asm volatile(
				"{\n"
				".reg .pred p;\n"
				".reg .b64 db;\n"
				"setp.ne.b32 p, %5, 0;\n"
				"mov.b64 db, {%2, %3};\n"
				"tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n"
				"}\n" ::"r"(d),
				"r"(a_tmem), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(add)
				: "memory");
		}
		// Shared-memory descriptors, 128-byte swizzle.  Queries and k lie K-major (rows of 64 elements of head_dim, 8-row groups 1024
		// bytes apart).  v lies with head_dim contiguous although the product runs over keys: the same 8-row groups are then 1024
		// bytes apart along the product's K, and the next 64 columns of head_dim a panel further.
		constexpr uint32_t DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);
		__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lead) {
			return ((addr >> 4) & 0x3FFFu) | ((lead >> 4) << 16);
		}
		// f32 accumulators, M = 128; b_by_columns: B's N side is contiguous
		constexpr uint32_t instr_desc(int n, bool bf16, bool b_by_columns) {
			return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_by_columns ? 1u : 0u) << 16) | (static_cast<uint32_t>(n >> 3) << 17) |
				(static_cast<uint32_t>(TILE >> 4) << 24);
		}

		// What P V of a step waits for, all on one barrier: the chain's eight warps have left the weights, the other chain's eight have
		// taken the product before it (the chains share its buffer), and the two warps that watch the ring have seen its v tile (and
		// cleaned it) and the k tile of the scores issued behind it.  The issuing thread must not wait often: while products stream
		// their operands from shared memory, a look at a barrier there takes some 250 cycles.
		constexpr int P_ARRIVALS = 8 + 8 + 2;
		// A slot of the ring is free once the products that read it have run and both watching warps have seen its tile: they follow
		// every phase of every slot by its parity, and a warp that comes after the slot's next tile would wait for a phase that has passed.
		constexpr int EMPTY_ARRIVALS = 1 + 2;
		__device__ __forceinline__ void mbar_arrive_n(uint64_t* bar, int n) {
			asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(n) : "memory");
		}

		// (a, b) in PARTS 16-bit parts
		template<bool BF16> __device__ __forceinline__ void split_parts(float a, float b, uint32_t (&p)[parts_of(BF16)]) {
			split2<BF16>(a, b, p[0], p[1]);
			if constexpr (BF16) {
				const __nv_bfloat162 h = *reinterpret_cast<const __nv_bfloat162*>(&p[0]), l = *reinterpret_cast<const __nv_bfloat162*>(&p[1]);
				const __nv_bfloat162 r = __floats2bfloat162_rn((a - __low2float(h)) - __low2float(l), (b - __high2float(h)) - __high2float(l));
				p[2]				   = *reinterpret_cast<const uint32_t*>(&r);
			}
		}

		// The same for weights (positive, at most 2^WEIGHT_BITS), by cutting bits off instead of rounding: a cut float converts exactly, so nothing
		// has to be converted back to find what is left.  bf16: 8 + 8 + 8 bits are the whole float; f16: 11 + 11 bits, off by at most
		// 2^-21 (below 2^-14, where f16 becomes subnormal, by at most 2^-25, i.e. 2^-39 of the largest weight).
		template<bool BF16> __device__ __forceinline__ void cut_parts(float a, float b, uint32_t (&p)[parts_of(BF16)]) {
			if constexpr (BF16) {
				p[0]		  = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
				const float x = a - __uint_as_float(__float_as_uint(a) & 0xffff0000u), y = b - __uint_as_float(__float_as_uint(b) & 0xffff0000u);
				p[1]		  = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
				const float u = x - __uint_as_float(__float_as_uint(x) & 0xffff0000u), v = y - __uint_as_float(__float_as_uint(y) & 0xffff0000u);
				p[2]		  = __byte_perm(__float_as_uint(u), __float_as_uint(v), 0x7632);
			} else {
				const float x	= __uint_as_float(__float_as_uint(a) & 0xffffe000u), y = __uint_as_float(__float_as_uint(b) & 0xffffe000u);
				float lx, ly;
				unpack2(fma2(pack2(x, y), pack2(-1.f, -1.f), pack2(a, b)), lx, ly);
				const __half2 h = __floats2half2_rn(x, y), l = __floats2half2_rn(lx, ly);
				p[0] = *reinterpret_cast<const uint32_t*>(&h);
				p[1] = *reinterpret_cast<const uint32_t*>(&l);
			}
		}

		__device__ __forceinline__ void softmax_barrier() {
			asm volatile("bar.sync 1, 512;" ::: "memory");
		}
		__device__ __forceinline__ void chain_barrier(int chain) {
			asm volatile("bar.sync %0, 256;" ::"r"(2 + chain) : "memory");
		}

		// The largest score of this thread's COLS columns from ts on.  CUT: columns past `left` are not seen.
		template<int COLS, bool CUT> __device__ __forceinline__ float tile_max(uint32_t ts, int left) {
			float t4[4] = { -INFINITY, -INFINITY, -INFINITY, -INFINITY };
#pragma unroll
			for (int ch = 0; ch < COLS / 16; ++ch) {
				uint32_t x[16];
				tmem_ld16(ts + ch * 16, x);
				tmem_ld_wait16(x);
#pragma unroll
				for (int i = 0; i < 16; i += 2) {
					float a = __uint_as_float(x[i]), b = __uint_as_float(x[i + 1]);
					if constexpr (CUT) {
						if (ch * 16 + i > left)
							a = -INFINITY;
						if (ch * 16 + i + 1 > left)
							b = -INFINITY;
					}
					t4[(i >> 1) & 3] = fmaxf(t4[(i >> 1) & 3], fmaxf(a, b));
				}
			}
			return fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3]));
		}
		// The scores become weights in place: parts 0 and 1 of 16 keys over their 16 scores, part 2 at t3.  Returns their sum.
		template<int COLS, bool BF16, bool CUT> __device__ __forceinline__ float tile_weights(uint32_t ts, uint32_t t3, int left, float factor, float bias) {
			constexpr int PARTS = parts_of(BF16);
			const uint64_t factor2 = pack2(factor, factor), bias2 = pack2(bias, bias);
			uint64_t s2 = pack2(0.f, 0.f);
#pragma unroll
			for (int ch = 0; ch < COLS / 16; ++ch) {
				uint32_t x[16], part[PARTS][8];
				tmem_ld16(ts + ch * 16, x);
				tmem_ld_wait16(x);
#pragma unroll
				for (int i = 0; i < 8; ++i) {
					float a = __uint_as_float(x[2 * i]), b = __uint_as_float(x[2 * i + 1]);
					if constexpr (CUT) {
						if (ch * 16 + 2 * i > left)
							a = -INFINITY;
						if (ch * 16 + 2 * i + 1 > left)
							b = -INFINITY;
					}
					unpack2(fma2(pack2(a, b), factor2, bias2), a, b);
					a  = ex2(a);
					b  = ex2(b);
					s2 = add2(s2, pack2(a, b));
					uint32_t q[PARTS];
					cut_parts<BF16>(a, b, q);
#pragma unroll
					for (int z = 0; z < PARTS; ++z)
						part[z][i] = q[z];
				}
				tmem_st8(ts + ch * 16, part[0]);
				tmem_st8(ts + ch * 16 + 8, part[1]);
				if constexpr (PARTS > 2)
					tmem_st8(t3 + ch * 8, part[2]);
			}
			float sa, sb;
			unpack2(s2, sa, sb);
			return sa + sb;
		}

		// The order in which the products need the tiles: `ahead` key tiles, then value and key tiles in turn, then the values that are
		// left.  Position of key tile j's k and v in it, of n tiles:
		__device__ __forceinline__ int k_at(int j, int ahead) {
			return j + max(0, j - ahead + 1);
		}
		__device__ __forceinline__ int v_at(int j, int n, int ahead) {
			return j + min(ahead + j, n);
		}

		template<int D, bool BF16, bool TWO> __global__ void __launch_bounds__(PT, 1)
			attn_prompt_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ prompt_params p) {
			constexpr int PARTS = parts_of(BF16), NS = score_buffers(BF16), PANELS = D / 64;
			constexpr int NST = ring_slots(D, BF16, TWO), SLOT = slot_bytes(D), PANEL = KT * 128;
			constexpr int QTILE = TILE * D * 2, TILES = TWO ? 2 : 1;
			constexpr uint32_t COL_S = 0, COL_O = NS * KT, COL_P3 = NS * KT + D;
			static_assert(NS * KT + D + (PARTS > 2 ? NS * KT / 2 : 0) <= 512, "tensor memory");
			static_assert(NST >= 3, "a ring of three at least");
			extern __shared__ unsigned char smem_raw[];
			unsigned char* base	 = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
			unsigned char* ring	 = base + q_bytes(D, BF16, TWO);
			prompt_head* hd		 = reinterpret_cast<prompt_head*>(ring + NST * SLOT);
			const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
			const int group = p.a.group;
			static_assert(q_bytes(D, BF16, TWO) + NST * SLOT + sizeof(prompt_head) <= 227 * 1024, "shared memory");
			if (reinterpret_cast<unsigned char*>(hd + 1) > smem_raw + prompt_smem(D, BF16, TWO)) {
				pdl_wait_prior_grids();
				if (tid == 0)
					atomicCAS(p.c.status, DEV_OK, DEV_KV_SMEM);
				return;
			}

			if (tid == 0) {
				for (int s = 0; s < NST; ++s) {
					mbar_init(&hd->full[s], 1);
					mbar_init(&hd->empty[s], EMPTY_ARRIVALS);
				}
				for (int b = 0; b < NS; ++b) {
					mbar_init(&hd->s_full[b], 1);
					mbar_init(&hd->p_full[b], P_ARRIVALS);
				}
				mbar_init(&hd->o_full[0], 1);
				mbar_init(&hd->o_full[1], 1);
				mbar_init(&hd->q_full, 16);
				mbar_init(&hd->drain, 1);
				fence_mbar_init();
				hd->odd	  = 0;
				hd->entry = -1;
				hd->total = 0;
			}
			pdl_launch_dependents();
			pdl_wait_prior_grids();
			__syncthreads();

			// ---- what this CTA computes ----
			int kvh, seq, row0, rows, q_row, key0 = 0, n_keys, pos0 = 0, split = 0;
			if (p.splits > 0) {
				int x = blockIdx.x;
				kvh	  = x % p.c.kv_heads;
				x /= p.c.kv_heads;
				split = x % p.splits;
				row0  = (x / p.splits) * TILE * TILES;
				rows  = min(TILE * TILES, p.a.M * group - row0);
				q_row = 0;
				// the first entry that is not padding lends its table
				for (int i = tid; i < p.a.n; i += PT)
					if (p.a.seqs[i] != -1)
						atomicMin(reinterpret_cast<unsigned*>(&hd->entry), static_cast<unsigned>(i));
				__syncthreads();
				const int e = hd->entry;
				seq			= e >= 0 ? p.a.seqs[e] : -1;
				if (seq < 0 || seq >= p.c.max_seqs)
					return;// reported by the decode kernel
				key0   = split * p.tiles_per_split * KT;
				n_keys = min(p.a.shared_pages << p.c.page_shift, key0 + p.tiles_per_split * KT);
			} else {
				// tiles of all list entries, in order; the CTAs take them from the end, where the causal rows with the most keys lie
				const auto tiles_of = [&](int i, bool tell) {
					const int s = p.a.seqs[i];
					if (s == -1)
						return 0;
					const int a = p.a.cu[i], b = p.a.cu[i + 1];
					if (s < 0 || s >= p.c.max_seqs || a < 0 || b < a || b > p.a.M || p.c.lens[s] < 0 || p.c.lens[s] > kv_capacity(p.c)) {
						if (tell)
							atomicCAS(p.c.status, DEV_OK, DEV_KV_BAD);
						return 0;
					}
					return static_cast<int>((static_cast<long long>(b - a) * group + TILE * TILES - 1) / (TILE * TILES));
				};
				// the grid holds the tiles of M rows; entries that name the same rows (cu falls behind a padding entry) can have more
				const auto check_grid = [&](int total) {
					if (blockIdx.x == 0 && tid == 0 && static_cast<long long>(total) * p.c.kv_heads > gridDim.x)
						atomicCAS(p.c.status, DEV_OK, DEV_KV_BAD);
				};
				kvh				 = blockIdx.x % p.c.kv_heads;
				const int rank	 = blockIdx.x / p.c.kv_heads;
				const bool short_list = p.a.n <= PT;// one look at the list does
				int total		 = 0;
				if (!short_list) {
					int mine = 0;
					for (int i = tid; i < p.a.n; i += PT)
						mine += tiles_of(i, blockIdx.x == 0);
					mine = __reduce_add_sync(0xffffffffu, mine);
					if (lane == 0 && mine)
						atomicAdd(&hd->total, mine);
					__syncthreads();
					total = hd->total;
					if (rank >= total)
						return;
					check_grid(total);
				}
				int before = 0;
				for (int i0 = 0; i0 < p.a.n; i0 += PT) {
					const int i = i0 + tid;
					const int t = i < p.a.n ? tiles_of(i, short_list && blockIdx.x == 0) : 0;
					int x		= t;
#pragma unroll
					for (int o = 1; o < 32; o <<= 1) {
						const int y = __shfl_up_sync(0xffffffffu, x, o);
						if (lane >= o)
							x += y;
					}
					if (lane == 31)
						hd->scan[warp] = x;
					__syncthreads();
					int sum = before, all = before;
					for (int w = 0; w < PT / 32; ++w) {
						const int y = hd->scan[w];
						sum += w < warp ? y : 0;
						all += y;
					}
					if (short_list) {
						total = all;
						if (rank >= total)
							return;
						check_grid(total);
					}
					const int want = total - 1 - rank;
					if (want >= sum + x - t && want < sum + x) {
						hd->tile  = want - (sum + x - t);
						hd->seq	  = p.a.seqs[i];
						hd->q_row = p.a.cu[i];
						hd->count = p.a.cu[i + 1] - p.a.cu[i];
						hd->len	  = p.c.lens[hd->seq];
					}
					before = all;
					__syncthreads();
					if (before > want)
						break;
				}
				seq				= hd->seq;
				q_row			= hd->q_row;
				const int count = hd->count;
				row0		= hd->tile * TILE * TILES;
				rows		= static_cast<int>(min(static_cast<long long>(TILE * TILES), static_cast<long long>(count) * group - row0));
				pos0		= hd->len - count;
				n_keys		= max(0, pos0 + (row0 + rows - 1) / group + 1);// as many as the last row sees
			}
			const int n_tiles = n_keys > key0 ? (n_keys - key0 + KT - 1) / KT : 0;
			const bool two	  = TWO && rows > TILE;
			// the first row's last key: tiles from `masked` on reach past it
			const int low	 = p.splits > 0 ? n_keys - 1 : pos0 + row0 / group;
			const int masked = low + 1 <= key0 ? 0 : (low + 1 - key0) / KT;
			const int steps	 = two ? 2 * n_tiles : n_tiles;// a step: one tile's keys for one chain
			const int ahead	 = two ? NS - 1 : NS;// key tiles whose scores are under way before the first P V

			if (warp == 1)
				tmem_alloc(&hd->tmem, 512);
			tc_fence_before();
			__syncthreads();
			tc_fence_after();
			const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&hd->tmem);

			if (warp < 4) {
				// launched with 640 x 96 registers: 128 x 32 + 512 x 112 are exactly those, 128 x 56 + 512 x 104 fit.  With 64 running sums a
				// thread needs the 112 (8192 tokens 871 us, with 104 911), with 32 the issuing warps the 56 (11 packed prompts 293 us, 331)
				if constexpr (D == 128)
					asm volatile("setmaxnreg.dec.sync.aligned.u32 32;" ::: "memory");
				else
					asm volatile("setmaxnreg.dec.sync.aligned.u32 56;" ::: "memory");
				if (warp == 0) {
					// ---------------- copies ----------------
					const int box	 = min(p.c.page_tokens, 64);
					const int pages	 = (n_keys + p.c.page_tokens - 1) >> p.c.page_shift;
					const int* row	 = p.c.table + static_cast<size_t>(seq) * p.c.max_pages;
					// one table cache for k and one for v: they are at different tiles
					int page[2] = { 0, 0 }, page0[2] = { -64, -64 };
					const int loads	 = 2 * n_tiles;
					bool ok			 = true;
					int issued		 = 0;
					int kj = 0, vj = 0;
					for (int at = 0; at < loads && ok; ++at) {
						const int is_v = !(kj < n_tiles && kj < ahead + vj);
						const int j	   = is_v ? vj++ : kj++;
						const int s		 = at % NST;
						const int k0	 = key0 + j * KT;
						const int boxes	 = (min(KT, n_keys - k0) + box - 1) / box;
						const int j0	= k0 >> p.c.page_shift;
						int number = is_v ? page[1] : page[0], from = is_v ? page0[1] : page0[0];
						if (j0 + ((boxes * box - 1) >> p.c.page_shift) >= from + 32) {
							from   = j0;
							number = j0 + lane < pages ? row[j0 + lane] : 0;
							if (number < 0 || number >= p.c.n_pages) {
								atomicCAS(p.c.status, DEV_OK, DEV_KV_BAD);
								number = 0;
							}
							if (is_v) {
								page[1]	 = number;
								page0[1] = from;
							} else {
								page[0]	 = number;
								page0[0] = from;
							}
						}
						if (lane == 0) {
							if (!mbar_wait(&hd->empty[s], ((at / NST) & 1) ^ 1)) {
								atomicExch(p.c.status, DEV_TIMEOUT_EMPTY);
								ok = false;
							} else {
								mbar_expect_tx(&hd->full[s], boxes * PANELS * box * 128);
							}
						}
						ok = __shfl_sync(0xffffffffu, ok, 0);
						// a lane per copy: box and panel of head_dim
						const int b = lane / PANELS, c = lane % PANELS;
						const int k	  = k0 + b * box;
						const int pg  = __shfl_sync(0xffffffffu, number, ((k >> p.c.page_shift) - from) & 31);
						if (b < boxes && ok)
							tma_load_2d(smem_u32(ring) + s * SLOT + c * PANEL + b * box * 128, is_v ? &map_v : &map_k, c * 64,
								((pg * p.c.kv_heads + kvh) << p.c.page_shift) + (k & (p.c.page_tokens - 1)), &hd->full[s]);
						issued += ok;
						__syncwarp();
					}
					// the last copy into each slot has landed before the block ends
					if (lane == 0)
						for (int at = max(0, issued - NST); at < issued; ++at)
							if (!mbar_wait(&hd->full[at % NST], (at / NST) & 1))
								atomicExch(p.c.status, DEV_TIMEOUT_DRAIN);
				} else if (warp == 1) {
					// ---------------- products ----------------
					if (elect_one() && n_tiles > 0) {
						constexpr uint32_t id_s = instr_desc(KT, BF16, false), id_o = instr_desc(D, BF16, true);
						const uint32_t ring_a = smem_u32(ring), q_a = smem_u32(base);
						bool ok = mbar_wait(&hd->q_full, 0);
						// whether the slot of this position of the ring's order is filled once more: nobody waits for it otherwise
						const auto again  = [&](int pos) { return pos + NST < 2 * n_tiles; };
						const auto scores = [&](int t) {
							const int c = t & 1, j = two ? t >> 1 : t, buf = t % NS, pos = k_at(j, ahead), s = pos % NST;
							const uint32_t d  = tmem + COL_S + buf * KT;
							const uint32_t kd = desc_lo(ring_a + s * SLOT, 16);
#pragma unroll
							for (int part = PARTS - 1; part >= 0; --part) {// the small parts first, while the truncating accumulator is small
								const uint32_t qd = desc_lo(q_a + (part * TILES + (two ? c : 0)) * QTILE, 16);
#pragma unroll
								for (int k = 0; k < D / 16; ++k)
									mma_ss(d, qd + (k >> 2) * ((TILE * 128) >> 4) + (k & 3) * 2, DESC_HI, kd + (k >> 2) * (PANEL >> 4) + (k & 3) * 2, DESC_HI, id_s, part < PARTS - 1 || k > 0);
							}
							umma_commit_a(smem_u32(&hd->s_full[buf]));
							if ((!two || c == 1) && again(pos))
								umma_commit_a(smem_u32(&hd->empty[s]));
						};
						// step t is chain t & 1; its scores are NS steps ahead, so their buffer is free once P V of step t - NS has been issued
						for (int t = 0; t < NS && t < steps && ok; ++t) {
							const int at = k_at(two ? t >> 1 : t, ahead);
							ok			 = mbar_wait(&hd->full[at % NST], (at / NST) & 1);
							tc_fence_after();
							if (ok)
								scores(t);
						}
						for (int t = 0; t < steps && ok; ++t) {
							const int c = t & 1, j = two ? t >> 1 : t, buf = t % NS, pos = v_at(j, n_tiles, ahead), s = pos % NST;
							ok = mbar_wait(&hd->p_full[buf], (t / NS) & 1);
							if (!ok)
								break;
							tc_fence_after();
							const uint32_t d  = tmem + COL_O;
							const uint32_t pw = tmem + COL_S + buf * KT, p3 = tmem + COL_P3 + buf * (KT / 2);
							const uint32_t vd = desc_lo(ring_a + s * SLOT, PANEL);
#pragma unroll
							for (int part = PARTS - 1; part >= 0; --part)
#pragma unroll
								for (int k = 0; k < KT / 16; ++k) {
									// 16 keys' weights sit in the 16 columns of their scores: 8 columns each of the first two parts
									const uint32_t w = part < 2 ? pw + k * 16 + part * 8 : p3 + k * 8;
									mma_ts(d, w, vd + k * (2048 >> 4), DESC_HI, id_o, part < PARTS - 1 || k > 0);
								}
							umma_commit_a(smem_u32(&hd->o_full[c]));
							if ((!two || c == 1) && again(pos))
								umma_commit_a(smem_u32(&hd->empty[s]));
							if (t + NS < steps)
								scores(t + NS);
						}
						if (!ok)
							atomicExch(p.c.status, DEV_TIMEOUT_MMA);
						umma_commit_a(smem_u32(&hd->drain));
						if (!mbar_wait(&hd->drain, 0))
							atomicExch(p.c.status, DEV_TIMEOUT_DRAIN);
					}
				} else {
					// ---------------- the ring's tiles, in order; v tiles that not every row sees whole are cleaned ----------------
					bool odd = false, ok = true;
					int seen = 0;// positions of the ring's order that have landed; the slot is not filled again before its arrival here
					const auto see = [&](int at) {
						for (; seen <= at && ok; ++seen) {
							ok = __all_sync(0xffffffffu, mbar_wait(&hd->full[seen % NST], (seen / NST) & 1));
							if (ok && lane == 0)
								mbar_arrive(&hd->empty[seen % NST]);
						}
					};
					for (int t = 0; t < steps && ok; ++t) {
						const int j = two ? t >> 1 : t, at = v_at(j, n_tiles, ahead), s = at % NST;
						see(at);
						unsigned char* v = ring + s * SLOT;
						const int k0	 = key0 + j * KT;
						const bool clean = j >= masked && (!two || (t & 1) == 0);
						// 8 lanes per row and panel
						for (int r = (warp - 2) * 4 + (lane >> 3); r < KT && ok && clean; r += 8) {
							if (k0 + r <= low)
								continue;
							const bool past = k0 + r >= n_keys;
#pragma unroll
							for (int c = 0; c < PANELS; ++c) {
								uint4* x = reinterpret_cast<uint4*>(v + c * PANEL + r * 128) + (lane & 7);
								if (past) {
									*x = make_uint4(0, 0, 0, 0);
									continue;
								}
								uint4 y		 = *x;
								uint32_t* w	 = &y.x;
								bool changed = false;
								constexpr uint32_t E = BF16 ? 0x7f80u : 0x7c00u;// the exponent of infinities and NaN
#pragma unroll
								for (int i = 0; i < 4; ++i) {
									if ((w[i] & E) == E) {
										w[i] &= 0xffff0000u;
										changed = true;
									}
									if ((w[i] & (E << 16)) == (E << 16)) {
										w[i] &= 0x0000ffffu;
										changed = true;
									}
								}
								if (changed) {
									*x	= y;
									odd = true;
								}
							}
						}
						if (odd)
							atomicExch(&hd->odd, 1);
						if (clean)
							fence_proxy_async();
						if (t + NS < steps)
							see(k_at(two ? (t + NS) >> 1 : t + NS, ahead));
						if (t >= NS && ok)// not ahead of the buffer's step before: an arrival would count for that one
							ok = __all_sync(0xffffffffu, mbar_wait(&hd->p_full[t % NS], (t / NS - 1) & 1));
						__syncwarp();
						if (lane == 0 && ok)// nothing was multiplied before step 0: no product to be taken
							mbar_arrive_n(&hd->p_full[t % NS], t == 0 && warp == 2 ? 1 + 8 : 1);
					}
					if (!ok && lane == 0)
						atomicExch(p.c.status, DEV_TIMEOUT_FULL);
				}
			} else {
				if constexpr (D == 128)
					asm volatile("setmaxnreg.inc.sync.aligned.u32 112;" ::: "memory");
				else
					asm volatile("setmaxnreg.inc.sync.aligned.u32 104;" ::: "memory");
				// two threads per row: one for each half of a tile's columns and of head_dim
				const int w16 = warp - 4, chain = w16 >> 3, half = (w16 >> 2) & 1;
				const int lrow = (w16 & 3) * 32 + lane;// row of the tile = lane of tensor memory
				// ---- queries: split a row (f16: scaled by a power of two), store the parts swizzled; D / 4 lanes per row ----
				{
					constexpr int LANES = D / 4, AT_ONCE = 32 / LANES;
					const int n_rows = two ? 2 * TILE : TILE;
					const int sub = lane / LANES, l4 = lane % LANES;
					constexpr int BATCH = 8;// loads in flight per lane
					for (int r0 = w16 * AT_ONCE; r0 < n_rows; r0 += 16 * AT_ONCE * BATCH) {
						float4 v[BATCH];
						int rr[BATCH];
#pragma unroll
						for (int i = 0; i < BATCH; ++i) {
							rr[i]		= r0 + i * 16 * AT_ONCE + sub;
							v[i]		= make_float4(0.f, 0.f, 0.f, 0.f);
							const int r = row0 + rr[i];
							if (rr[i] < rows && rr[i] < n_rows)
								v[i] = __ldg(reinterpret_cast<const float4*>(p.a.q + (q_row + static_cast<long long>(r / group)) * p.a.ldq + static_cast<long long>(kvh * group + r % group) * D) + l4);
						}
#pragma unroll
						for (int i = 0; i < BATCH; ++i) {
							float f = 1.f, back = 1.f;
							if constexpr (!BF16) {
								float amax = fmaxf(fmaxf(fabsf(v[i].x), fabsf(v[i].y)), fmaxf(fabsf(v[i].z), fabsf(v[i].w)));
#pragma unroll
								for (int o = LANES / 2; o > 0; o >>= 1)
									amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
								f = row_scaling(amax, &back);
							}
							if (rr[i] < n_rows) {
								uint32_t a[PARTS], b[PARTS];
								split_parts<BF16>(v[i].x * f, v[i].y * f, a);
								split_parts<BF16>(v[i].z * f, v[i].w * f, b);
								const int r = rr[i] & (TILE - 1), t = rr[i] / TILE;
								const int chunk = (l4 >> 1) & 7, panel = l4 >> 4;
								const int off	= panel * (TILE * 128) + r * 128 + ((chunk ^ (r & 7)) << 4) + (l4 & 1) * 8;
#pragma unroll
								for (int part = 0; part < PARTS; ++part)
									*reinterpret_cast<uint2*>(base + (part * TILES + t) * QTILE + off) = make_uint2(a[part], b[part]);
								if (l4 == 0)
									hd->back[rr[i]] = back * p.a.scale2;
							}
						}
					}
					fence_proxy_async();
					__syncwarp();
					if (lane == 0)
						mbar_arrive(&hd->q_full);
					softmax_barrier();
				}
				const int crow	   = two ? chain * TILE + lrow : lrow;// row of the CTA
				const float factor = hd->back[crow];
				softmax_barrier();// the space is the chains' from here on
				const int r		   = row0 + crow;
				const int token	   = r / group;
				const int last	   = crow >= rows ? -1 : (p.splits > 0 ? n_keys - 1 : pos0 + token);// the last key this row sees
				constexpr int COLS = KT / 2, DIMS = D / 2;
				const int d0	   = half * DIMS;// this thread's part of head_dim
				const uint32_t at  = tmem + (static_cast<uint32_t>((w16 & 3) * 32) << 16);
				const uint32_t to = at + COL_O + d0;
				float o[DIMS];
#pragma unroll
				for (int d = 0; d < DIMS; ++d)
					o[d] = 0.f;
				float m = -INFINITY, l = 0.f;
				bool ok	= true;
				int use = 0;
				// the product of this chain's tile `n` joins the running sums, which `keep` brings to the tile's maximum
				const auto add_product = [&](int n, float keep) {
					ok = ok && mbar_wait(&hd->o_full[chain], n & 1);
					tc_fence_after();
#pragma unroll
					for (int ch = 0; ch < DIMS / 16; ++ch) {
						uint32_t x[16];
						tmem_ld16(to + ch * 16, x);
						tmem_ld_wait16(x);
#pragma unroll
						for (int i = 0; i < 16; ++i)
							o[ch * 16 + i] = fmaf(o[ch * 16 + i], keep, __uint_as_float(x[i]));
					}
					tc_fence_before();
					__syncwarp();
					if (lane == 0 && ok && 2 * n + chain + 1 < steps)
						mbar_arrive(&hd->p_full[(2 * n + chain + 1) % NS]);
				};
				for (int j = two ? 0 : chain; j < n_tiles; j += two ? 1 : 2, ++use) {
					const int step = 2 * use + chain, buf = step % NS;
					const uint32_t ts = at + COL_S + buf * KT + half * COLS, t3 = at + COL_P3 + buf * (KT / 2) + half * (COLS / 2);
					ok = ok && mbar_wait(&hd->s_full[buf], (step / NS) & 1);
					tc_fence_after();
					const bool cut = j >= masked;
					const int left = last - (key0 + j * KT) - half * COLS;// columns 0 .. left of this half are seen
					// (no way out of the loop between the barriers: all threads of the chain take part in every one)
					hd->half[chain][half][lrow] = cut ? tile_max<COLS, true>(ts, left) : tile_max<COLS, false>(ts, left);
					chain_barrier(chain);
					const float top	 = fmaxf(m, fmaxf(hd->half[chain][0][lrow], hd->half[chain][1][lrow]) * factor);
					const float mm	 = top == -INFINITY ? 0.f : top;
					const float keep = ex2(m - mm);
					m				 = top;
					const float sum	 = cut ? tile_weights<COLS, BF16, true>(ts, t3, left, factor, WEIGHT_BITS<BF16> - mm) : tile_weights<COLS, BF16, false>(ts, t3, left, factor, WEIGHT_BITS<BF16> - mm);
					tmem_st_wait();
					tc_fence_before();
					__syncwarp();
					if (lane == 0 && ok)
						mbar_arrive(&hd->p_full[buf]);
					l = fmaf(l, keep, sum);
					add_product(use, keep);
				}
				if (!ok)
					atomicExch(p.c.status, DEV_TIMEOUT_MMA);
				tc_fence_before();
				softmax_barrier();// all products have run, all maxima are read
				hd->half[chain][half][lrow] = l;
				const bool joined = !two && n_tiles > 1;// (with one tile the second chain had nothing to do)
				if (joined && chain == 1) {
					// odd key tiles into even ones, through the space of the queries
					float* mo = reinterpret_cast<float*>(base);// [D][128]
#pragma unroll
					for (int d = 0; d < DIMS; ++d)
						mo[(d0 + d) * TILE + lrow] = o[d];
					reinterpret_cast<float*>(ring)[half * TILE + lrow] = m;
				}
				softmax_barrier();
				l = hd->half[chain][0][lrow] + hd->half[chain][1][lrow];
				if (joined && chain == 0) {
					const float* mo = reinterpret_cast<const float*>(base);
					const float m1 = reinterpret_cast<const float*>(ring)[half * TILE + lrow], l1 = hd->half[1][0][lrow] + hd->half[1][1][lrow];
					const float top = fmaxf(m, m1), mm = top == -INFINITY ? 0.f : top;
					const float f0 = ex2(m - mm), f1 = ex2(m1 - mm);
					l = l * f0 + l1 * f1;
					m = top;
#pragma unroll
					for (int d = 0; d < DIMS; ++d)
						o[d] = fmaf(mo[(d0 + d) * TILE + lrow], f1, o[d] * f0);
				}
				if ((two || chain == 0) && crow < rows) {
					if (*reinterpret_cast<volatile int*>(&hd->odd)) {
						// infinities and NaN that were taken out of v: back for the rows that see them
						const int* table = p.c.table + static_cast<size_t>(seq) * p.c.max_pages;
						for (int k = max(key0, low + 1); k <= last; ++k) {
							const int pg = table[k >> p.c.page_shift];
							if (pg < 0 || pg >= p.c.n_pages)
								continue;
							const uint32_t* v = reinterpret_cast<const uint32_t*>(p.c.v + static_cast<size_t>(p.a.layer) * p.c.layer_bytes +
								((((static_cast<size_t>(pg) * p.c.kv_heads + kvh) << p.c.page_shift) + (k & (p.c.page_tokens - 1))) * D + d0) * 2);
#pragma unroll
							for (int i = 0; i < DIMS / 2; ++i) {
								const uint32_t w = v[i];
								float a, b;
								if constexpr (BF16) {
									a = __uint_as_float(w << 16);
									b = __uint_as_float(w & 0xffff0000u);
								} else {
									const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
									a			   = f.x;
									b			   = f.y;
								}
								if (!(fabsf(a) < INFINITY))
									o[2 * i] += a;
								if (!(fabsf(b) < INFINITY))
									o[2 * i + 1] += b;
							}
						}
					}
					if (p.splits > 0) {
						const long long part = (static_cast<long long>(kvh) * p.splits + split) * (static_cast<long long>(p.a.M) * group) + r;
						float4* dst			 = reinterpret_cast<float4*>(p.o + part * D + d0);
#pragma unroll
						for (int d = 0; d < DIMS / 4; ++d)
							__stcg(dst + d, make_float4(o[4 * d], o[4 * d + 1], o[4 * d + 2], o[4 * d + 3]));
						if (half == 0)
							__stcg(p.ml + part, make_float2(m, l));
					} else {
						const float inv = last >= 0 ? 1.f / l : 0.f;
						float4* dst = reinterpret_cast<float4*>(p.a.out + (q_row + static_cast<long long>(token)) * p.a.ldo + static_cast<long long>(kvh * group + r - token * group) * D + d0);
#pragma unroll
						for (int d = 0; d < DIMS / 4; ++d)
							dst[d] = make_float4(o[4 * d] * inv, o[4 * d + 1] * inv, o[4 * d + 2] * inv, o[4 * d + 3] * inv);
					}
				}
			}
			tc_fence_before();
			__syncthreads();
			if (warp == 1) {
				tc_fence_after();
				tmem_dealloc(tmem, 512);
			}
		}

		// The splits of a prefix become one, in place of the first: a warp per row and kv head.  (Read by the decode kernel split by split,
		// in the short pieces of a batch, they cost it 30 us where this launch takes 4.)
		template<int D> __global__ void __launch_bounds__(256) attn_prefix_join_kernel(float* __restrict__ o, float2* __restrict__ ml, int rows, int splits, int kv_heads) {
			constexpr int V = D / 32, FLY = 8;// columns of a lane, splits in flight
			pdl_launch_dependents();
			pdl_wait_prior_grids();
			const int lane = threadIdx.x & 31;
			for (long long y = (blockIdx.x * 256ll + threadIdx.x) >> 5; y < static_cast<long long>(rows) * kv_heads; y += gridDim.x * 8ll) {
				const long long kvh = y / rows, first = kvh * splits * rows + (y - kvh * rows);
				float m = -INFINITY, l = 0.f, acc[V] = {};
				for (int s0 = 0; s0 < splits; s0 += FLY) {
					float2 x[FLY];
					float v[FLY][V];
#pragma unroll
					for (int j = 0; j < FLY; ++j) {
						const long long at = first + static_cast<long long>(min(s0 + j, splits - 1)) * rows;
						x[j]			   = __ldcg(ml + at);
#pragma unroll
						for (int i = 0; i < V; i += 2) {
							const float2 w = __ldcg(reinterpret_cast<const float2*>(o + at * D + lane * V + i));
							v[j][i]		   = w.x;
							v[j][i + 1]	   = w.y;
						}
					}
					float top = m;
#pragma unroll
					for (int j = 0; j < FLY; ++j)
						top = fmaxf(top, x[j].x);
					const float mm = top == -INFINITY ? 0.f : top, keep = ex2(m - mm);
					m = top;
					l *= keep;
#pragma unroll
					for (int i = 0; i < V; ++i)
						acc[i] *= keep;
#pragma unroll
					for (int j = 0; j < FLY; ++j)
						if (s0 + j < splits) {
							const float f = ex2(x[j].x - mm);
							l			  = fmaf(x[j].y, f, l);
#pragma unroll
							for (int i = 0; i < V; ++i)
								acc[i] = fmaf(v[j][i], f, acc[i]);
						}
				}
#pragma unroll
				for (int i = 0; i < V; i += 2)
					*reinterpret_cast<float2*>(o + first * D + lane * V + i) = make_float2(acc[i], acc[i + 1]);
				__syncwarp();// every lane has read the row's (maximum, sum)
				if (lane == 0)
					ml[first] = make_float2(m, l);
			}
		}

		typedef void (*prompt_kernel_t)(const CUtensorMap, const CUtensorMap, const prompt_params);
		prompt_kernel_t pick_kernel(int d, bool bf16, bool two, int* smem) {
			*smem = prompt_smem(d, bf16, two);
			if (d == 128)
				return bf16 ? attn_prompt_kernel<128, true, false> : (two ? attn_prompt_kernel<128, false, true> : attn_prompt_kernel<128, false, false>);
			if (bf16)
				return two ? attn_prompt_kernel<64, true, true> : attn_prompt_kernel<64, true, false>;
			return two ? attn_prompt_kernel<64, false, true> : attn_prompt_kernel<64, false, false>;
		}

		int launch_prompt_kernel(nhb_ctx* ctx, const prompt_params& p, bool two, long long grid) {
			CUtensorMap mk, mv;
			if (!make_page_map(&mk, p.c, p.c.k, p.a.layer) || !make_page_map(&mv, p.c, p.c.v, p.a.layer))
				return fail(ctx, NHB_ERR_CUDA, "attention: cuTensorMapEncodeTiled failed");
			if (grid > INT32_MAX)
				return fail(ctx, NHB_ERR_UNSUPPORTED, "attention: more than 2^31 - 1 tiles");
			int smem			 = 0;
			prompt_kernel_t kern = pick_kernel(p.c.head_dim, p.c.bf16 != 0, two, &smem);
			if (int rc = kv_allow_smem(ctx, reinterpret_cast<const void*>(kern), smem); rc != NHB_OK)
				return rc;
			cudaError_t e = kv_launch(ctx, kern, dim3(static_cast<unsigned>(grid)), dim3(PT), smem, mk, mv, p);
			return e == cudaSuccess ? NHB_OK : fail_cuda(ctx, e, "attn_prompt launch");
		}

	}

	int launch_attn_prompt(nhb_ctx* ctx, const kv_view& c, const attn_args& a) {
		// Two row tiles per CTA where that still gives every SM a CTA (f16, 32 heads of 128 on 8, two against one: 700 tokens, 88 CTAs of
		// two, 40.9 / 34.3 us; 1000 tokens 52.0 / 46.1; 2048 tokens, 256 CTAs, 101.6 / 114.3; 4096 tokens 283 / 291)
		const long long rows = static_cast<long long>(a.M) * a.group;
		const bool two		 = two_fits(c.head_dim, c.bf16 != 0) && rows / (2 * TILE) * c.kv_heads >= ctx->sm_count;
		prompt_params p{};
		p.c = c;
		p.a = a;
		// no fewer tiles than the list can hold: every entry may leave one partly filled
		return launch_prompt_kernel(ctx, p, two, (rows / (two ? 2 * TILE : TILE) + a.n) * c.kv_heads);
	}

	// How the keys that a batch shares are dealt: row tiles x kv heads x splits make about one CTA per SM, and two row tiles per CTA read a
	// split's keys once
	prefix_plan plan_prefix(const nhb_ctx* ctx, const kv_view& c, const attn_args& a) {
		prefix_plan r{};
		const int kt		 = KT;
		const long long keys = static_cast<long long>(a.shared_pages) << c.page_shift;
		const long long rows = static_cast<long long>(a.M) * a.group;
		r.two				 = two_fits(c.head_dim, c.bf16 != 0) && rows > TILE;
		r.row_tiles			 = (rows + (r.two ? 2 : 1) * TILE - 1) / ((r.two ? 2 : 1) * TILE);
		const int tiles		 = static_cast<int>((keys + kt - 1) / kt);
		const long long ctas = r.row_tiles * c.kv_heads;
		const int want		 = static_cast<int>(std::max<long long>(1, ctx->sm_count / ctas));
		r.tiles_per_split	 = (tiles + want - 1) / std::max(1, want);
		if (r.tiles_per_split < 1)
			r.tiles_per_split = 1;
		r.splits = (tiles + r.tiles_per_split - 1) / r.tiles_per_split;
		const size_t parts = static_cast<size_t>(c.kv_heads) * r.splits * rows;
		r.bytes			   = parts * c.head_dim * sizeof(float) + parts * sizeof(float2);
		return r;
	}

	int launch_attn_prefix(nhb_ctx* ctx, const kv_view& c, const attn_args& a, const prefix_plan& plan, void* ws, attn_prefix* out) {
		prompt_params p{};
		p.c				   = c;
		p.a				   = a;
		p.splits		   = plan.splits;
		p.tiles_per_split  = plan.tiles_per_split;
		const size_t parts = static_cast<size_t>(c.kv_heads) * plan.splits * a.M * a.group;
		p.o				   = static_cast<float*>(ws);
		p.ml			   = reinterpret_cast<float2*>(p.o + parts * c.head_dim);
		out->o			   = p.o;
		out->ml			   = p.ml;
		out->any		   = 1;
		const int rows	   = a.M * a.group;
		out->stride		   = static_cast<long long>(plan.splits) * rows;
		const int rc	   = launch_prompt_kernel(ctx, p, plan.two, plan.row_tiles * plan.splits * c.kv_heads);
		if (rc != NHB_OK || plan.splits == 1)
			return rc;
		const dim3 grid(static_cast<unsigned>(std::min<long long>((static_cast<long long>(rows) * c.kv_heads + 7) / 8, 8ll * ctx->sm_count)));
		cudaError_t e = kv_launch(ctx, c.head_dim == 128 ? attn_prefix_join_kernel<128> : attn_prefix_join_kernel<64>, grid, dim3(256), 0, p.o, p.ml, rows, plan.splits, c.kv_heads);
		return e == cudaSuccess ? NHB_OK : fail_cuda(ctx, e, "attn_prefix_join launch");
	}

}
