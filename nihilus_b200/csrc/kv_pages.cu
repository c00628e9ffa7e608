// Pages of the K/V cache: reserving, forking, freeing and compacting (the reference reserves [max_seq] rows per layer up front,
// include/nihilus-incl/infra/core_traits.hpp:240-245, and has no counterpart).
//
// The bookkeeping -- tables, lengths, reference counts -- lives in device memory and is changed by kernels only, so that a step
// that opens new pages can be part of a captured graph.  Each call is decided as a whole by one CTA (what is needed, whether the
// request is sound, which free pages it gets) before anything changes; copies of page contents follow in a second, wide launch.
// "The lowest free pages, in the order of the list" makes the outcome a function of the state alone.
//
// Copies are bound by memory: 24 forks of the 8B model's cache (265 MB read and written) take 46 us with the freeing of the 24 before,
// a compaction that moves 19 pages of 8 MB 51 us (6.2 TB/s).  The small calls are bound by their launches, 3 to 4 us each in a graph.
#include "kv_cache.h"
#include "ptx.cuh"

namespace nhb {

	namespace {

		constexpr int PLAN_THREADS = 1024;
		constexpr int PER_THREAD   = 8;// reference counts a thread looks at per step of the search for free pages

		// first words of the workspace; then base[n], then the page lists
		struct plan_head {
			int ok;// the request is sound and there are pages for it
			int copies;// entries of src / dst / rows
			int live;// compaction: pages in use
			int pad[13];
		};
		struct plan_lists {
			plan_head* head;
			int* base;// [n] first entry of dst that belongs to list entry i
			int* dst;// [n_pages]
			int* src;// [n_pages]
			int* rows;// [n_pages] rows to copy
		};
		__host__ __device__ plan_lists lists_at(void* ws, long long n, int n_pages) {
			plan_lists l;
			l.head = static_cast<plan_head*>(ws);
			l.base = reinterpret_cast<int*>(l.head + 1);
			l.dst  = l.base + n;
			l.src  = l.dst + n_pages;
			l.rows = l.src + n_pages;
			return l;
		}
		size_t lists_bytes(long long n, int n_pages) {
			return sizeof(plan_head) + (static_cast<size_t>(n) + 3 * static_cast<size_t>(n_pages)) * sizeof(int);
		}

		__device__ __forceinline__ void report(int* status, int code) {
			atomicCAS(status, DEV_OK, code);
		}

		// exclusive sum of v over the block in thread order; *total the sum.  smem: 32 values.  All threads call it.
		template<typename T> __device__ T block_scan(T v, T* total, T* smem) {
			const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n_warps = blockDim.x >> 5;
			T x			   = v;
#pragma unroll
			for (int o = 1; o < 32; o <<= 1) {
				const T y = __shfl_up_sync(0xffffffffu, x, o);
				if (lane >= o)
					x += y;
			}
			__syncthreads();// smem of the call before is read
			if (lane == 31)
				smem[warp] = x;
			__syncthreads();
			if (warp == 0) {
				T w = lane < n_warps ? smem[lane] : 0;
#pragma unroll
				for (int o = 1; o < 32; o <<= 1) {
					const T y = __shfl_up_sync(0xffffffffu, w, o);
					if (lane >= o)
						w += y;
				}
				smem[lane] = w;
			}
			__syncthreads();
			*total = smem[n_warps - 1];
			return x - v + (warp ? smem[warp - 1] : 0);
		}

		// Writes the page numbers in [lo, hi) whose count is zero (want_free) or not, ascending, to out[0 .. most), where most is
		// what out can take.  Returns how many there are, up to `most` (the search stops there).
		__device__ int collect(const int* refs, int lo, int hi, bool want_free, int* out, int most, int* smem) {
			int found = 0;
			for (int p0 = lo; p0 < hi && found < most; p0 += PLAN_THREADS * PER_THREAD) {
				const int first = p0 + static_cast<int>(threadIdx.x) * PER_THREAD;
				unsigned mask	= 0;
#pragma unroll
				for (int j = 0; j < PER_THREAD; ++j)
					if (first + j < hi && (__ldcg(refs + first + j) == 0) == want_free)
						mask |= 1u << j;
				int total;
				int at = found + block_scan(__popc(mask), &total, smem);
				if (out)
#pragma unroll
					for (int j = 0; j < PER_THREAD; ++j)
						if (mask & (1u << j)) {
							if (at < most)
								out[at] = first + j;
							++at;
						}
				found += total;
			}
			return found < most ? found : most;
		}

		// marks sequence s in the bitmap; true if it was marked before
		__device__ __forceinline__ bool mark(unsigned* bits, int s) {
			return (atomicOr(bits + (s >> 5), 1u << (s & 31)) >> (s & 31)) & 1u;
		}

		// ---- reserve: one CTA ----
		__global__ void __launch_bounds__(PLAN_THREADS) kv_reserve_kernel(kv_view c, const int* __restrict__ seqs, const int* __restrict__ cu, int n, void* ws) {
			extern __shared__ unsigned bits[];// one bit per sequence
			__shared__ int scan[32];
			__shared__ long long wide_scan[32];
			pdl_launch_dependents();
			pdl_wait_prior_grids();
			const int refused  = __ldcg(c.status + KV_REFUSED);// (on its way beside the lookups)
			const plan_lists l = lists_at(ws, n, c.n_pages);
			const int tid	   = threadIdx.x;
			for (int i = tid; i < (c.max_seqs + 31) / 32; i += PLAN_THREADS)
				bits[i] = 0;
			__syncthreads();
			bool bad		= false;
			long long total = 0;// the needs of a sound request can add up to more than there are pages
			for (int i0 = 0; i0 < n; i0 += PLAN_THREADS) {
				const int i = i0 + tid;
				long long need = 0, sum;
				if (i < n) {
					const int s = seqs[i];
					if (s != -1) {
						if (s < -1 || s >= c.max_seqs || mark(bits, s)) {
							bad = true;
						} else {
							const int count = cu ? cu[i + 1] - cu[i] : 1;
							const int old	= c.lens[s];
							if (count < 0 || old < 0 || old > kv_capacity(c) || count > kv_capacity(c) - old)
								bad = true;
							else
								need = kv_pages_of(c, old + count) - kv_pages_of(c, old);
						}
					}
				}
				const long long at = block_scan(need, &sum, wide_scan);
				if (i < n)
					l.base[i] = static_cast<int>(total + at);// only read where the total fits
				total += sum;
			}
			if (__syncthreads_or(bad) || refused) {
				if (tid == 0 && !refused) {
					report(c.status, DEV_KV_BAD);
					c.status[KV_REFUSED] = 1;
				}
				return;
			}
			// (most decode steps open no page at all and skip the search)
			if (total > c.n_pages || (total > 0 && collect(c.refs, 0, c.n_pages, true, l.dst, static_cast<int>(total), scan) < total)) {
				if (tid == 0) {
					report(c.status, DEV_KV_NO_PAGES);
					c.status[KV_REFUSED] = 1;
				}
				return;
			}
			__syncthreads();// base and dst are written
			const int lane = tid & 31;
			for (int i = tid >> 5; i < n; i += PLAN_THREADS / 32) {
				const int s = seqs[i];
				if (s == -1)
					continue;
				const int old	= c.lens[s];
				const int now	= old + (cu ? cu[i + 1] - cu[i] : 1);
				const int first = kv_pages_of(c, old), need = kv_pages_of(c, now) - first;
				int* row		= c.table + static_cast<size_t>(s) * c.max_pages + first;
				for (int j = lane; j < need; j += 32) {
					const int page = l.dst[l.base[i] + j];
					row[j]		   = page;
					c.refs[page]   = 1;
				}
				__syncwarp();
				if (lane == 0)
					c.lens[s] = now;
			}
		}

		// ---- fork: the plan (one CTA), then tables and copies ----
		__global__ void __launch_bounds__(PLAN_THREADS) kv_fork_plan_kernel(kv_view c, const int* __restrict__ parents, const int* __restrict__ children, int n, int deep,
			void* ws) {
			extern __shared__ unsigned bits[];// one bit per sequence: children, then parents that have been looked at
			__shared__ int scan[32];
			__shared__ long long wide_scan[32];
			pdl_launch_dependents();
			pdl_wait_prior_grids();
			const plan_lists l = lists_at(ws, n, c.n_pages);
			const int tid	   = threadIdx.x;
			for (int i = tid; i < 2 * ((c.max_seqs + 31) / 32); i += PLAN_THREADS)
				bits[i] = 0;
			__syncthreads();
			bool bad		= false;
			long long total = 0;
			for (int i0 = 0; i0 < n; i0 += PLAN_THREADS) {
				const int i = i0 + tid;
				long long need = 0, sum;
				if (i < n && children[i] != -1) {
					const int p = parents[i], s = children[i];
					if (s < -1 || s >= c.max_seqs || p < 0 || p >= c.max_seqs || mark(bits, s) || c.lens[s] != 0 || c.lens[p] < 0 || c.lens[p] > kv_capacity(c))
						bad = true;
					else
						need = deep ? kv_pages_of(c, c.lens[p]) : ((c.lens[p] & (c.page_tokens - 1)) != 0);
				}
				const long long at = block_scan(need, &sum, wide_scan);
				if (i < n)
					l.base[i] = static_cast<int>(total + at);
				total += sum;
			}
			__syncthreads();// all children are marked
			// a parent is nobody's child, and its table (looked at once, by a warp) holds pages only
			const int lane	 = tid & 31;
			unsigned* looked = bits + (c.max_seqs + 31) / 32;
			for (int i = tid >> 5; i < n; i += PLAN_THREADS / 32) {
				const int p = parents[i];
				if (children[i] == -1 || p < 0 || p >= c.max_seqs)
					continue;
				if ((bits[p >> 5] >> (p & 31)) & 1u)
					bad = true;
				const int tokens = c.lens[p];
				if (__shfl_sync(0xffffffffu, lane == 0 ? mark(looked, p) : false, 0) || tokens < 0 || tokens > kv_capacity(c))
					continue;
				const int* row = c.table + static_cast<size_t>(p) * c.max_pages;
				for (int j = lane; j < kv_pages_of(c, tokens); j += 32)
					if (row[j] < 0 || row[j] >= c.n_pages)
						bad = true;
			}
			if (__syncthreads_or(bad)) {
				if (tid == 0) {
					l.head->ok = 0;
					report(c.status, DEV_KV_BAD);
				}
				return;
			}
			if (total > c.n_pages || (total > 0 && collect(c.refs, 0, c.n_pages, true, l.dst, static_cast<int>(total), scan) < total)) {
				if (tid == 0) {
					l.head->ok = 0;
					report(c.status, DEV_KV_NO_PAGES);
				}
				return;
			}
			__syncthreads();
			for (int i = tid >> 5; i < n; i += PLAN_THREADS / 32) {
				if (children[i] == -1)
					continue;
				const int tokens = c.lens[parents[i]];
				const int held = kv_pages_of(c, tokens), first = deep ? 0 : tokens >> c.page_shift;
				const int* row = c.table + static_cast<size_t>(parents[i]) * c.max_pages;
				for (int j = first + lane; j < held; j += 32) {
					const int at	  = l.base[i] + j - first;
					l.src[at]		  = row[j];
					l.rows[at]		  = min(c.page_tokens, tokens - (j << c.page_shift));
					c.refs[l.dst[at]] = 1;
				}
			}
			if (tid == 0) {
				l.head->ok	   = 1;
				l.head->copies = static_cast<int>(total);
			}
		}

		// Copies rows [0, rows[i]) of page src[i] to page dst[i] for all layers, k and v, and kv heads.  A warp moves one head's rows
		// of one page (2 to 32 KB, contiguous) with 16-byte loads, eight in flight per lane.
		__device__ void copy_pages(const kv_view& c, const plan_lists& l, int copies, int warp, int n_warps, int lane) {
			const int row16			= c.head_dim >> 3;// 16-byte words of a row
			const long long head16	= static_cast<long long>(c.page_tokens) * row16;
			const long long page16	= head16 * c.kv_heads;
			const long long layer16 = page16 * c.n_pages;
			const int per_copy		= c.n_layers * 2 * c.kv_heads;
			const long long tasks	= static_cast<long long>(copies) * per_copy;
			for (long long t = warp; t < tasks; t += n_warps) {
				const int i		= static_cast<int>(t / per_copy);
				int r			= static_cast<int>(t - static_cast<long long>(i) * per_copy);
				const int h		= r % c.kv_heads;
				r /= c.kv_heads;
				uint4* pool		  = reinterpret_cast<uint4*>((r & 1) ? c.v : c.k) + (r >> 1) * layer16 + h * head16;
				const uint4* from = pool + __ldcg(l.src + i) * page16;
				uint4* to		  = pool + __ldcg(l.dst + i) * page16;
				const int words	  = __ldcg(l.rows + i) * row16;
				for (int w0 = lane; w0 < words; w0 += 32 * 8) {
					uint4 v[8];
#pragma unroll
					for (int j = 0; j < 8; ++j)
						if (w0 + 32 * j < words)
							v[j] = __ldcs(from + w0 + 32 * j);
#pragma unroll
					for (int j = 0; j < 8; ++j)
						if (w0 + 32 * j < words)
							__stcs(to + w0 + 32 * j, v[j]);
				}
			}
		}

		__global__ void __launch_bounds__(256) kv_fork_apply_kernel(kv_view c, const int* __restrict__ parents, const int* __restrict__ children, int n, int deep, void* ws) {
			pdl_launch_dependents();
			pdl_wait_prior_grids();
			const plan_lists l = lists_at(ws, n, c.n_pages);
			if (!__ldcg(&l.head->ok))
				return;
			for (int i = blockIdx.x; i < n; i += gridDim.x) {
				if (children[i] == -1)
					continue;
				const int tokens = c.lens[parents[i]];// parents are nobody's children: nobody writes their lengths here
				const int held = kv_pages_of(c, tokens), shared = deep ? 0 : tokens >> c.page_shift;
				const int* from = c.table + static_cast<size_t>(parents[i]) * c.max_pages;
				int* row		= c.table + static_cast<size_t>(children[i]) * c.max_pages;
				for (int j = threadIdx.x; j < c.max_pages; j += blockDim.x) {
					int page = -1;
					if (j < shared) {
						page = from[j];
						atomicAdd(c.refs + page, 1);
					} else if (j < held) {
						page = __ldcg(l.dst + __ldcg(l.base + i) + j - shared);
					}
					row[j] = page;
				}
				if (threadIdx.x == 0)
					c.lens[children[i]] = tokens;
			}
			copy_pages(c, l, __ldcg(&l.head->copies), (blockIdx.x * blockDim.x + threadIdx.x) >> 5, (gridDim.x * blockDim.x) >> 5, threadIdx.x & 31);
		}

		// ---- free: every CTA checks the whole list (same answer everywhere), then ends its share of the sequences ----
		__global__ void __launch_bounds__(256) kv_free_kernel(kv_view c, const int* __restrict__ seqs, int n) {
			extern __shared__ unsigned bits[];
			pdl_launch_dependents();
			pdl_wait_prior_grids();
			for (int i = threadIdx.x; i < (c.max_seqs + 31) / 32; i += blockDim.x)
				bits[i] = 0;
			__syncthreads();
			bool bad = false;
			for (int i = threadIdx.x; i < n; i += blockDim.x) {
				const int s = seqs[i];
				if (s != -1 && (s < -1 || s >= c.max_seqs || mark(bits, s)))
					bad = true;
			}
			if (__syncthreads_or(bad)) {
				if (blockIdx.x == 0 && threadIdx.x == 0)
					report(c.status, DEV_KV_BAD);
				return;
			}
			for (int i = blockIdx.x; i < n; i += gridDim.x) {
				const int s = seqs[i];
				if (s == -1)
					continue;
				const int tokens = c.lens[s];
				const bool sound = tokens >= 0 && tokens <= kv_capacity(c);
				const int held	 = sound ? kv_pages_of(c, tokens) : 0;
				int* row		 = c.table + static_cast<size_t>(s) * c.max_pages;
				if (!sound && threadIdx.x == 0)
					report(c.status, DEV_KV_BAD);
				for (int j = threadIdx.x; j < c.max_pages; j += blockDim.x) {
					if (j < held) {
						const int page = row[j];
						if (page >= 0 && page < c.n_pages)
							atomicSub(c.refs + page, 1);
						else
							report(c.status, DEV_KV_BAD);
					}
					row[j] = -1;
				}
				__syncthreads();// every thread has the length
				if (threadIdx.x == 0)
					c.lens[s] = 0;
			}
		}

		// ---- compact ----
		__global__ void __launch_bounds__(PLAN_THREADS) kv_compact_plan_kernel(kv_view c, int* __restrict__ live_out, void* ws) {
			__shared__ int scan[32];
			pdl_launch_dependents();
			pdl_wait_prior_grids();
			const plan_lists l = lists_at(ws, 0, c.n_pages);
			bool bad		   = false;// a length that its table row cannot hold: the sequence's pages would move without it
			for (int s = threadIdx.x; s < c.max_seqs; s += PLAN_THREADS)
				bad = bad || c.lens[s] < 0 || c.lens[s] > kv_capacity(c);
			const int live = collect(c.refs, 0, c.n_pages, false, nullptr, c.n_pages, scan);
			if (__syncthreads_or(bad)) {
				if (threadIdx.x == 0) {
					l.head->copies = 0;
					report(c.status, DEV_KV_BAD);
				}
				return;
			}
			// as many pages in use above `live` as free ones below it
			const int moves = collect(c.refs, 0, live, true, l.dst, c.n_pages, scan);
			__syncthreads();
			if (moves)
				collect(c.refs, live, c.n_pages, false, l.src, moves, scan);
			__syncthreads();
			// rows: which move a page takes part in, by its old number (what the others hold there is no move of theirs)
			for (int i = threadIdx.x; i < moves; i += PLAN_THREADS) {
				const int from = l.src[i], to = l.dst[i];
				l.rows[from] = i;
				c.refs[to]	 = c.refs[from];
				c.refs[from] = 0;
			}
			if (threadIdx.x == 0) {
				l.head->copies = moves;
				l.head->live   = live;
				if (live_out)
					*live_out = live;
			}
		}

		__global__ void __launch_bounds__(256) kv_compact_apply_kernel(kv_view c, void* ws) {
			pdl_launch_dependents();
			pdl_wait_prior_grids();
			const plan_lists l = lists_at(ws, 0, c.n_pages);
			const int moves	   = __ldcg(&l.head->copies);
			if (moves == 0)
				return;
			const int live = __ldcg(&l.head->live);
			const int warp = (blockIdx.x * blockDim.x + threadIdx.x) >> 5, n_warps = (gridDim.x * blockDim.x) >> 5, lane = threadIdx.x & 31;
			for (int s = warp; s < c.max_seqs; s += n_warps) {
				const int held = kv_pages_of(c, c.lens[s]);
				int* row	   = c.table + static_cast<size_t>(s) * c.max_pages;
				for (int j = lane; j < held; j += 32) {
					const int page = row[j];
					if (page < 0 || page >= c.n_pages) {
						report(c.status, DEV_KV_BAD);
					} else if (page >= live) {
						const int move = __ldcg(l.rows + page);
						if (move >= 0 && move < moves && __ldcg(l.src + move) == page)
							row[j] = __ldcg(l.dst + move);
						else
							report(c.status, DEV_KV_BAD);// nobody counts the page
					}
				}
			}
			// whole pages: [kv_heads][page_tokens][head_dim] is one stretch of memory, moved in pieces of 4 KB
			const long long page16	= (static_cast<long long>(c.kv_heads) * c.page_tokens * c.head_dim) >> 3;
			const long long layer16 = page16 * c.n_pages;
			const int pieces		= static_cast<int>((page16 + 255) / 256);
			const int per_copy		= c.n_layers * 2 * pieces;
			const long long tasks	= static_cast<long long>(moves) * per_copy;
			for (long long t = warp; t < tasks; t += n_warps) {
				const int i		  = static_cast<int>(t / per_copy);
				int r			  = static_cast<int>(t - static_cast<long long>(i) * per_copy);
				const int piece	  = r % pieces;
				r /= pieces;
				uint4* pool		  = reinterpret_cast<uint4*>((r & 1) ? c.v : c.k) + (r >> 1) * layer16 + piece * 256;
				const uint4* from = pool + __ldcg(l.src + i) * page16;
				uint4* to		  = pool + __ldcg(l.dst + i) * page16;
				const int words	  = static_cast<int>(min(256ll, page16 - piece * 256ll));
				uint4 v[8];
#pragma unroll
				for (int j = 0; j < 8; ++j)
					if (lane + 32 * j < words)
						v[j] = __ldcs(from + lane + 32 * j);
#pragma unroll
				for (int j = 0; j < 8; ++j)
					if (lane + 32 * j < words)
						__stcs(to + lane + 32 * j, v[j]);
			}
		}

		// CTAs of eight warps for at most `tasks` pieces of copying and `rows` table rows, up to eight per SM: a small call does not pay for
		// the launch of a thousand
		unsigned copy_grid(const nhb_ctx* ctx, double tasks, long long rows) {
			const double want = std::max(tasks / 8, static_cast<double>(rows));
			return static_cast<unsigned>(std::max(1.0, std::min(want, 8.0 * ctx->sm_count)));
		}

		size_t bitmap_bytes(const kv_view& c) {
			return static_cast<size_t>((c.max_seqs + 31) / 32) * 4;
		}

	}

	// ---- checks and workspace, shared by the cache's operators ----
	int check_cache(nhb_ctx* ctx, const nhb_kv_cache* cache, kv_view* out, const char* who) {
		const std::string w(who);
		if (!cache)
			return fail(ctx, NHB_ERR_ARG, w + ": null cache");
		if (cache->type != NHB_KV_F16 && cache->type != NHB_KV_BF16)
			return fail(ctx, NHB_ERR_ARG, w + ": unknown cache type");
		if (cache->head_dim != 64 && cache->head_dim != 128)
			return fail(ctx, NHB_ERR_UNSUPPORTED, w + ": head_dim must be 64 or 128");
		if (cache->page_tokens != 16 && cache->page_tokens != 32 && cache->page_tokens != 64 && cache->page_tokens != 128)
			return fail(ctx, NHB_ERR_UNSUPPORTED, w + ": page_tokens must be 16, 32, 64 or 128");
		if (cache->n_layers < 1 || cache->n_layers > 65536 || cache->n_pages < 1 || cache->n_pages > NHB_KV_MAX_PAGES || cache->kv_heads < 1 || cache->kv_heads > 1024 ||
			cache->max_seqs < 1 || cache->max_seqs > NHB_KV_MAX_SEQS || cache->max_pages < 1 || cache->max_pages > (int64_t(1) << 30) / cache->page_tokens)
			return fail(ctx, NHB_ERR_ARG, w + ": a size of the cache is out of range (layers and sequences up to 65536, pages up to 2^24, kv heads up to 1024, 2^30 tokens per sequence)");
		if (cache->n_pages * cache->kv_heads * cache->page_tokens > INT32_MAX)
			return fail(ctx, NHB_ERR_UNSUPPORTED, w + ": more than 2^31 - 1 rows (pages x kv heads x page_tokens) in a layer");
		if (!cache->k || !cache->v || !cache->table || !cache->lens || !cache->refs)
			return fail(ctx, NHB_ERR_ARG, w + ": null pointer in the cache");
		if (((reinterpret_cast<uintptr_t>(cache->k) | reinterpret_cast<uintptr_t>(cache->v)) & 15) ||
			((reinterpret_cast<uintptr_t>(cache->table) | reinterpret_cast<uintptr_t>(cache->lens) | reinterpret_cast<uintptr_t>(cache->refs)) & 3))
			return fail(ctx, NHB_ERR_ARG, w + ": misaligned pointer in the cache (k and v 16-byte aligned)");
		out->k			 = static_cast<char*>(cache->k);
		out->v			 = static_cast<char*>(cache->v);
		out->table		 = cache->table;
		out->lens		 = cache->lens;
		out->refs		 = cache->refs;
		out->n_layers	 = static_cast<int>(cache->n_layers);
		out->n_pages	 = static_cast<int>(cache->n_pages);
		out->kv_heads	 = static_cast<int>(cache->kv_heads);
		out->page_tokens = static_cast<int>(cache->page_tokens);
		out->page_shift	 = cache->page_tokens == 16 ? 4 : (cache->page_tokens == 32 ? 5 : (cache->page_tokens == 64 ? 6 : 7));
		out->head_dim	 = static_cast<int>(cache->head_dim);
		out->max_seqs	 = static_cast<int>(cache->max_seqs);
		out->max_pages	 = static_cast<int>(cache->max_pages);
		out->bf16		 = cache->type == NHB_KV_BF16;
		out->status		 = ctx ? ctx->dev_status : nullptr;
		out->layer_bytes = cache->n_pages * cache->kv_heads * cache->page_tokens * cache->head_dim * 2;
		return NHB_OK;
	}

	int check_layer(nhb_ctx* ctx, const kv_view& c, int64_t layer, const char* who) {
		if (layer < 0 || layer >= c.n_layers)
			return fail(ctx, NHB_ERR_ARG, std::string(who) + ": no such layer in the cache");
		return NHB_OK;
	}

	int check_rows(nhb_ctx* ctx, const float* p, int64_t ld, int64_t width, const char* who, const char* what) {
		if (!p || (reinterpret_cast<uintptr_t>(p) & 15) || ld < width || (ld & 3))
			return fail(ctx, NHB_ERR_ARG, std::string(who) + ": " + what + ": null or misaligned rows (16-byte aligned, leading dimension at least the row length and a multiple of 4)");
		return NHB_OK;
	}

	int check_list(nhb_ctx* ctx, const int32_t* seqs, const int32_t* cu, int64_t n, const char* who) {
		if (n < 0 || n > NHB_KV_MAX_SEQS)
			return fail(ctx, NHB_ERR_ARG, std::string(who) + ": 0 to 65536 list entries");
		if (n > 0 && (!seqs || (reinterpret_cast<uintptr_t>(seqs) & 3) || (reinterpret_cast<uintptr_t>(cu) & 3)))
			return fail(ctx, NHB_ERR_ARG, std::string(who) + ": null or misaligned list");
		return NHB_OK;
	}

	bool rows_overlap(const float* a, int64_t lda, int64_t wa, int64_t ma, const float* b, int64_t ldb, int64_t wb, int64_t mb) {
		if (ma < 1 || mb < 1)
			return false;
		if (!(a < b + (mb - 1) * ldb + wb && b < a + (ma - 1) * lda + wa))
			return false;
		if (lda == ldb) {
			// columns of one buffer side by side (q, k and v behind a joint projection) do not meet although their ranges do
			const int64_t d = ((b - a) % lda + lda) % lda;
			return !(d >= wa && d + wb <= lda);
		}
		return true;
	}

	int kv_workspace(nhb_ctx* ctx, size_t bytes, void** out, const char* who) {
		cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
		NHB_CUDA(ctx, cudaStreamIsCapturing(ctx->stream, &st));
		if (st == cudaStreamCaptureStatusNone) {
			if (int rc = kv_workspace_use(ctx); rc != NHB_OK)
				return rc;
		} else {
			// (a capture runs nothing now; its replays are ordered by nhb_graph_launch, or by the caller for a capture of the caller's own)
			ctx->kv_ws_captured = true;
		}
		bytes += NHB_KV_COUNTER_BYTES;
		if (bytes > ctx->kv_ws_cap) {
			if (ctx->capturing || st != cudaStreamCaptureStatusNone)
				return fail(ctx, NHB_ERR_UNSUPPORTED, std::string(who) + ": the workspace must grow during graph capture; run the same calls once before it");
			const size_t want = (std::max(bytes, 2 * ctx->kv_ws_cap) + (size_t(1) << 20) - 1) & ~((size_t(1) << 20) - 1);
			void* p			  = nullptr;
			cudaError_t e	  = cudaMalloc(&p, want);
			if (e == cudaErrorMemoryAllocation) {
				cudaGetLastError();
				return fail(ctx, NHB_ERR_NOMEM, std::string(who) + ": no device memory for the workspace");
			}
			if (e == cudaSuccess)
				e = cudaMemsetAsync(p, 0, NHB_KV_COUNTER_BYTES, ctx->stream);
			if (e != cudaSuccess) {
				if (p)
					cudaFree(p);
				return fail_cuda(ctx, e, "K/V workspace");
			}
			if (ctx->kv_ws)
				ctx->kv_ws_old.push_back(ctx->kv_ws);
			ctx->kv_ws	   = p;
			ctx->kv_ws_cap = want;
		}
		*out = static_cast<char*>(ctx->kv_ws) + NHB_KV_COUNTER_BYTES;
		return NHB_OK;
	}

	void kv_workspace_mark(nhb_ctx* ctx) {
		if (!ctx->kv_ws_busy || !ctx->kv_ws_unmarked)
			return;
		// (the query fails for the legacy stream while another stream's capture keeps it from being used: the event comes later)
		cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
		cudaError_t e			   = cudaStreamIsCapturing(ctx->kv_ws_stream, &st);
		if (e == cudaSuccess && st == cudaStreamCaptureStatusNone) {
			if (!ctx->kv_ws_ev)
				e = cudaEventCreateWithFlags(&ctx->kv_ws_ev, cudaEventDisableTiming);
			if (e == cudaSuccess)
				e = cudaEventRecord(ctx->kv_ws_ev, ctx->kv_ws_stream);
			if (e == cudaSuccess) {
				ctx->kv_ws_unmarked = false;
				ctx->kv_ws_stream	= nullptr;// the stream may end, and another one be given its handle: the next use waits, whatever its stream
			}
		}
		if (e != cudaSuccess)
			cudaGetLastError();
	}

	int kv_workspace_use(nhb_ctx* ctx) {
		if (ctx->kv_ws_busy && ctx->kv_ws_stream != ctx->stream) {
			kv_workspace_mark(ctx);
			if (ctx->kv_ws_unmarked)
				return fail(ctx, NHB_ERR_UNSUPPORTED, "the K/V workspace was last used on a stream that cannot be waited for now (it is being captured)");
			NHB_CUDA(ctx, cudaStreamWaitEvent(ctx->stream, ctx->kv_ws_ev, 0));
		}
		ctx->kv_ws_stream = ctx->stream;
		ctx->kv_ws_busy = ctx->kv_ws_unmarked = true;
		return NHB_OK;
	}

}

using namespace nhb;

extern "C" {

int nhb_kv_reserve(nhb_ctx* ctx, const nhb_kv_cache* cache, const int32_t* seqs_dev, const int32_t* cu_dev, int64_t n) {
	const char* who = "nhb_kv_reserve";
	kv_view c;
	int rc = check_cache(ctx, cache, &c, who);
	if (rc == NHB_OK)
		rc = check_list(ctx, seqs_dev, cu_dev, n, who);
	if (rc == NHB_OK && !ctx)
		rc = fail(ctx, NHB_ERR_ARG, std::string(who) + ": null context");
	if (rc != NHB_OK || n == 0)
		return rc;
	device_guard g(ctx->device);
	void* ws = nullptr;
	rc		 = kv_workspace(ctx, lists_bytes(n, c.n_pages), &ws, who);
	if (rc == NHB_OK)
		rc = wait_pending(ctx);
	if (rc != NHB_OK)
		return rc;
	cudaError_t e = kv_launch(ctx, kv_reserve_kernel, dim3(1), dim3(PLAN_THREADS), bitmap_bytes(c), c, seqs_dev, cu_dev, static_cast<int>(n), ws);
	return e == cudaSuccess ? NHB_OK : fail_cuda(ctx, e, "kv_reserve launch");
}

int nhb_kv_fork(nhb_ctx* ctx, const nhb_kv_cache* cache, const int32_t* parents_dev, const int32_t* children_dev, int64_t n, int deep) {
	const char* who = "nhb_kv_fork";
	kv_view c;
	int rc = check_cache(ctx, cache, &c, who);
	if (rc == NHB_OK)
		rc = check_list(ctx, parents_dev, nullptr, n, who);
	if (rc == NHB_OK)
		rc = check_list(ctx, children_dev, nullptr, n, who);
	if (rc == NHB_OK && !ctx)
		rc = fail(ctx, NHB_ERR_ARG, std::string(who) + ": null context");
	if (rc != NHB_OK || n == 0)
		return rc;
	device_guard g(ctx->device);
	void* ws = nullptr;
	rc		 = kv_workspace(ctx, lists_bytes(n, c.n_pages), &ws, who);
	if (rc == NHB_OK)
		rc = wait_pending(ctx);
	if (rc != NHB_OK)
		return rc;
	const int dp  = deep != 0;
	cudaError_t e = kv_launch(ctx, kv_fork_plan_kernel, dim3(1), dim3(PLAN_THREADS), 2 * bitmap_bytes(c), c, parents_dev, children_dev, static_cast<int>(n), dp, ws);
	if (e == cudaSuccess)
		e = kv_launch(ctx, kv_fork_apply_kernel, dim3(copy_grid(ctx, static_cast<double>(n) * (dp ? c.max_pages : 1) * c.n_layers * 2 * c.kv_heads, n)), dim3(256), 0, c, parents_dev, children_dev, static_cast<int>(n), dp, ws);
	return e == cudaSuccess ? NHB_OK : fail_cuda(ctx, e, "kv_fork launch");
}

int nhb_kv_free(nhb_ctx* ctx, const nhb_kv_cache* cache, const int32_t* seqs_dev, int64_t n) {
	const char* who = "nhb_kv_free";
	kv_view c;
	int rc = check_cache(ctx, cache, &c, who);
	if (rc == NHB_OK)
		rc = check_list(ctx, seqs_dev, nullptr, n, who);
	if (rc == NHB_OK && !ctx)
		rc = fail(ctx, NHB_ERR_ARG, std::string(who) + ": null context");
	if (rc != NHB_OK || n == 0)
		return rc;
	device_guard g(ctx->device);
	rc = wait_pending(ctx);
	if (rc != NHB_OK)
		return rc;
	const int grid = static_cast<int>(std::min<int64_t>(n, ctx->sm_count));
	cudaError_t e  = kv_launch(ctx, kv_free_kernel, dim3(grid), dim3(256), bitmap_bytes(c), c, seqs_dev, static_cast<int>(n));
	return e == cudaSuccess ? NHB_OK : fail_cuda(ctx, e, "kv_free launch");
}

int nhb_kv_compact(nhb_ctx* ctx, const nhb_kv_cache* cache, int32_t* live_dev) {
	const char* who = "nhb_kv_compact";
	kv_view c;
	int rc = check_cache(ctx, cache, &c, who);
	if (rc != NHB_OK)
		return rc;
	if (reinterpret_cast<uintptr_t>(live_dev) & 3)
		return fail(ctx, NHB_ERR_ARG, "nhb_kv_compact: misaligned pointer");
	if (!ctx)
		return fail(ctx, NHB_ERR_ARG, "nhb_kv_compact: null context");
	device_guard g(ctx->device);
	void* ws = nullptr;
	rc		 = kv_workspace(ctx, lists_bytes(0, c.n_pages), &ws, who);
	if (rc == NHB_OK)
		rc = wait_pending(ctx);
	if (rc != NHB_OK)
		return rc;
	cudaError_t e = kv_launch(ctx, kv_compact_plan_kernel, dim3(1), dim3(PLAN_THREADS), 0, c, live_dev, ws);
	if (e == cudaSuccess)
		e = kv_launch(ctx, kv_compact_apply_kernel,
			dim3(copy_grid(ctx, 0.5 * c.n_pages * c.n_layers * 2 * ((static_cast<double>(c.kv_heads) * c.page_tokens * c.head_dim) / 2048 + 1), (c.max_seqs + 7) / 8)), dim3(256), 0, c, ws);
	return e == cudaSuccess ? NHB_OK : fail_cuda(ctx, e, "kv_compact launch");
}
}
