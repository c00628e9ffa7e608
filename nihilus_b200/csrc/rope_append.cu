// Rotary embedding of q and k, and the store of k and v into the pages of the cache: the rope and cache-store nodes between the
// projections and the attention (include/nihilus-incl/infra/core_traits.hpp:577-618; the reference's kernels are empty).
//
// One CTA per token.  The angle position * base^(-2i/dims) / factor is formed in 64 bits, in turns, and reduced to [-1/2, 1/2] before
// it is rounded to 32: 64 threads make the token's 64 pairs of cos and sin once, and all heads read them from shared memory (in
// every head anew they would cost more than the rows' traffic).  The rest is a stream: 8 elements of a head per thread, two
// 16-byte loads, one or two stores.  Bytes per token: 8 per q element, 6 per k and v element.  B200: 2149 tokens of 32 + 8 heads of 128
// 21.4 us (4.5 TB/s), 64 tokens 4.0 us.  (Slower: reading rows before the
// token's place is known, 23.9 us; four tokens per CTA, which halves the lookups and the CTAs that hide them, 28.0.)
#include <cmath>

#include <cuda_bf16.h>

#include "kv_cache.h"
#include "ptx.cuh"

namespace nhb {

	namespace {

		constexpr int ROPE_THREADS = 256;

		struct rope_table {
			double turns[64];// turns per position of pair i: base^(-2i/dims) / 2 pi
			const float* factors;
			int dims;// 0: no rotation
			int halves;
		};

		struct append_args {
			const float *q, *k, *v;
			float* q_out;
			long long ldq, ldk, ldv, ldqo;
			const int *seqs, *cu;
			int n, heads, layer;
		};

		__device__ __forceinline__ uint32_t pack16(float lo, float hi, int bf16) {
			if (bf16) {
				const __nv_bfloat162 r = __floats2bfloat162_rn(lo, hi);
				return *reinterpret_cast<const uint32_t*>(&r);
			}
			const __half2 r = __floats2half2_rn(lo, hi);
			return *reinterpret_cast<const uint32_t*>(&r);
		}

		// which list entry token t belongs to: cu[e] <= t < cu[e + 1] (the first such entry where the list is not ascending); -1: none.  All threads call it.
		__device__ int entry_of(const int* cu, int n, int t, int* slot) {
			if (!cu)
				return t < n ? t : -1;
			if (threadIdx.x == 0)
				*slot = INT32_MAX;
			__syncthreads();
			for (int i = threadIdx.x; i < n; i += ROPE_THREADS)
				if (cu[i] <= t && t < cu[i + 1])
					atomicMin(slot, i);
			__syncthreads();
			return *slot == INT32_MAX ? -1 : *slot;
		}

		__global__ void __launch_bounds__(ROPE_THREADS) rope_kv_append_kernel(kv_view c, append_args a, rope_table r) {
			__shared__ float2 turn[64];// cos, sin
			__shared__ int slot;
			pdl_launch_dependents();
			pdl_wait_prior_grids();
			const int t = blockIdx.x, tid = threadIdx.x;
			const int refused = __ldcg(c.status + KV_REFUSED);// (on its way beside the lookups)
			const int e = entry_of(a.cu, a.n, t, &slot);
			if (e < 0)
				return;
			const int s = a.seqs[e];
			if (s == -1 || refused)
				return;
			// the position, and where the token's rows of the cache lie; a token the table has no page for is reported and skipped
			bool sound	   = s >= 0 && s < c.max_seqs;
			const int len  = sound ? c.lens[s] : 0;
			const int pos  = a.cu ? len - (a.cu[e + 1] - t) : len - 1;
			sound		   = sound && pos >= 0 && len <= kv_capacity(c);
			const int page = sound ? c.table[static_cast<size_t>(s) * c.max_pages + (pos >> c.page_shift)] : -1;
			if (!sound || page < 0 || page >= c.n_pages) {
				if (tid == 0)
					atomicCAS(c.status, DEV_OK, DEV_KV_BAD);
				return;
			}
			const int pairs = r.dims >> 1;
			if (tid < pairs) {
				double x = static_cast<double>(pos) * r.turns[tid];
				if (r.factors)
					x = static_cast<double>(pos) * (r.turns[tid] / static_cast<double>(r.factors[tid]));
				float sn, cs;
				sincospif(2.f * static_cast<float>(x - rint(x)), &sn, &cs);
				turn[tid] = make_float2(cs, sn);
			}
			__syncthreads();
			const int D = c.head_dim, units = D >> 3;// 8 elements per thread
			const size_t row = ((static_cast<size_t>(page) * c.kv_heads) << c.page_shift) + (pos & (c.page_tokens - 1));// of kv head 0, in rows of D
			char* const kp	 = c.k + static_cast<size_t>(a.layer) * c.layer_bytes;
			char* const vp	 = c.v + static_cast<size_t>(a.layer) * c.layer_bytes;
			const int total	 = (a.heads + 2 * c.kv_heads) * units;
			for (int i = tid; i < total; i += ROPE_THREADS) {
				const int head = i / units, u = i - head * units;
				const bool is_q = head < a.heads, is_k = !is_q && head < a.heads + c.kv_heads;
				const int h		= is_q ? head : (is_k ? head - a.heads : head - a.heads - c.kv_heads);
				const float* src = (is_q ? a.q + t * a.ldq : (is_k ? a.k + t * a.ldk : a.v + t * a.ldv)) + static_cast<size_t>(h) * D;
				// the two groups of four elements this thread owns
				const bool turned = 8 * u < r.dims && (is_q || is_k);
				const bool apart  = turned && r.halves;
				const int d0 = apart ? 4 * u : 8 * u, d1 = apart ? d0 + pairs : d0 + 4;
				float4 x = *reinterpret_cast<const float4*>(src + d0), y = *reinterpret_cast<const float4*>(src + d1);
				if (apart) {
					float* xs = &x.x;
					float* ys = &y.x;
#pragma unroll
					for (int j = 0; j < 4; ++j) {
						const float2 w = turn[d0 + j];
						const float x0 = xs[j], y0 = ys[j];
						xs[j] = x0 * w.x - y0 * w.y;
						ys[j] = x0 * w.y + y0 * w.x;
					}
				} else if (turned) {
					const float2 w0 = turn[4 * u], w1 = turn[4 * u + 1], w2 = turn[4 * u + 2], w3 = turn[4 * u + 3];
					x = make_float4(x.x * w0.x - x.y * w0.y, x.x * w0.y + x.y * w0.x, x.z * w1.x - x.w * w1.y, x.z * w1.y + x.w * w1.x);
					y = make_float4(y.x * w2.x - y.y * w2.y, y.x * w2.y + y.y * w2.x, y.z * w3.x - y.w * w3.y, y.z * w3.y + y.w * w3.x);
				}
				if (is_q) {
					float* dst = a.q_out + t * a.ldqo + static_cast<size_t>(h) * D;
					*reinterpret_cast<float4*>(dst + d0) = x;
					*reinterpret_cast<float4*>(dst + d1) = y;
				} else {
					// rounded to the cache's 16 bits once, to nearest; values beyond its range become infinities as in any conversion
					char* dst = (is_k ? kp : vp) + ((row + (static_cast<size_t>(h) << c.page_shift)) * D) * 2;
					const uint2 lo = make_uint2(pack16(x.x, x.y, c.bf16), pack16(x.z, x.w, c.bf16));
					const uint2 hi = make_uint2(pack16(y.x, y.y, c.bf16), pack16(y.z, y.w, c.bf16));
					if (apart) {
						*reinterpret_cast<uint2*>(dst + d0 * 2) = lo;
						*reinterpret_cast<uint2*>(dst + d1 * 2) = hi;
					} else {
						*reinterpret_cast<uint4*>(dst + d0 * 2) = make_uint4(lo.x, lo.y, hi.x, hi.y);
					}
				}
			}
		}

	}

}

using namespace nhb;

extern "C" int nhb_rope_kv_append(nhb_ctx* ctx, const nhb_kv_cache* cache, int64_t layer, const float* q_dev, int64_t ldq, int64_t heads, const float* k_dev, int64_t ldk,
	const float* v_dev, int64_t ldv, int64_t M, const int32_t* seqs_dev, const int32_t* cu_dev, int64_t n, const nhb_rope* rope, float* q_out_dev, int64_t ldqo) {
	const char* who = "nhb_rope_kv_append";
	kv_view c;
	int rc = check_cache(ctx, cache, &c, who);
	if (rc == NHB_OK)
		rc = check_layer(ctx, c, layer, who);
	if (rc == NHB_OK)
		rc = check_list(ctx, seqs_dev, cu_dev, n, who);
	if (rc != NHB_OK)
		return rc;
	if (heads < 1 || heads > 65536 || M < 0 || M > (int64_t(1) << 24) || (!cu_dev && M > n))
		return fail(ctx, NHB_ERR_ARG, "nhb_rope_kv_append: heads 1 to 65536, M 0 to 2^24 and, without cu, at most one row per list entry");
	rope_table r{};
	if (rope) {
		if (!(rope->base > 0.0) || !std::isfinite(rope->base) || rope->dims < 8 || rope->dims > c.head_dim || rope->dims % 8 != 0 ||
			(rope->style != NHB_ROPE_PAIRS && rope->style != NHB_ROPE_HALVES) || (reinterpret_cast<uintptr_t>(rope->factors_dev) & 3))
			return fail(ctx, NHB_ERR_ARG, "nhb_rope_kv_append: bad rotation (base > 0, dims a multiple of 8 up to head_dim, a known style)");
		r.dims	  = static_cast<int>(rope->dims);
		r.halves  = rope->style == NHB_ROPE_HALVES;
		r.factors = rope->factors_dev;
		for (int i = 0; i < r.dims / 2; ++i)
			r.turns[i] = std::pow(rope->base, -2.0 * i / r.dims) / 6.283185307179586476925286766559;
	}
	if (M == 0 || n == 0)
		return ctx ? NHB_OK : fail(ctx, NHB_ERR_ARG, "nhb_rope_kv_append: null context");
	const int64_t qw = heads * c.head_dim, kw = static_cast<int64_t>(c.kv_heads) * c.head_dim;
	if ((rc = check_rows(ctx, q_dev, ldq, qw, who, "q")) != NHB_OK || (rc = check_rows(ctx, k_dev, ldk, kw, who, "k")) != NHB_OK ||
		(rc = check_rows(ctx, v_dev, ldv, kw, who, "v")) != NHB_OK || (rc = check_rows(ctx, q_out_dev, ldqo, qw, who, "q_out")) != NHB_OK)
		return rc;
	const bool in_place = q_out_dev == q_dev && ldqo == ldq;
	if ((!in_place && rows_overlap(q_dev, ldq, qw, M, q_out_dev, ldqo, qw, M)) || rows_overlap(k_dev, ldk, kw, M, q_out_dev, ldqo, qw, M) ||
		rows_overlap(v_dev, ldv, kw, M, q_out_dev, ldqo, qw, M))
		return fail(ctx, NHB_ERR_ARG, "nhb_rope_kv_append: q_out overlaps an input (it may be q itself, with the same leading dimension)");
	if (!ctx)
		return fail(ctx, NHB_ERR_ARG, "nhb_rope_kv_append: null context");
	device_guard g(ctx->device);
	if ((rc = wait_pending(ctx)) != NHB_OK)
		return rc;
	append_args a{ q_dev, k_dev, v_dev, q_out_dev, ldq, ldk, ldv, ldqo, seqs_dev, cu_dev, static_cast<int>(n), static_cast<int>(heads), static_cast<int>(layer) };
	cudaError_t e = kv_launch(ctx, rope_kv_append_kernel, dim3(static_cast<unsigned>(M)), dim3(ROPE_THREADS), 0, c, a, r);
	return e == cudaSuccess ? NHB_OK : fail_cuda(ctx, e, "rope_kv_append launch");
}
