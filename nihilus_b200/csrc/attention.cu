// Entry points of the attention over the paged K/V cache: the attention core between the cache and attn_output
// (include/nihilus-incl/infra/core_traits.hpp:700-767; the reference's kernels are empty).  Host code; the kernels are in
// attn_prompt.cu (many rows on the tensor cores) and attn_decode.cu (one row per sequence, bound by the cache's bytes).
#include <cmath>

#include "attention.h"

namespace nhb {

	namespace {

		int run_attention(nhb_ctx* ctx, const nhb_kv_cache* cache, int64_t layer, const float* q, int64_t ldq, int64_t heads, int64_t M, const int32_t* seqs,
			const int32_t* cu, int64_t n, int64_t shared, float scale, float* out, int64_t ldo, const char* who) {
			kv_view c;
			int rc = check_cache(ctx, cache, &c, who);
			if (rc == NHB_OK)
				rc = check_layer(ctx, c, layer, who);
			if (rc == NHB_OK)
				rc = check_list(ctx, seqs, cu, n, who);
			if (rc != NHB_OK)
				return rc;
			if (heads < 1 || heads > 65536 || heads % c.kv_heads != 0 || M < 0 || M > (int64_t(1) << 24) || !(scale > 0.f) || !std::isfinite(scale))
				return fail(ctx, NHB_ERR_ARG, std::string(who) + ": heads a multiple of kv_heads, M 0 to 2^24, scale > 0");
			if (M == 0 || n == 0)
				return ctx ? NHB_OK : fail(ctx, NHB_ERR_ARG, std::string(who) + ": null context");
			if (M * (heads / c.kv_heads) > INT32_MAX - 1024)
				return fail(ctx, NHB_ERR_UNSUPPORTED, std::string(who) + ": too many rows (rows times query heads per kv head reach 2^31)");
			if (shared >> c.page_shift > c.max_pages)
				return fail(ctx, NHB_ERR_ARG, std::string(who) + ": more shared tokens than a sequence can hold");
			const int64_t w = heads * c.head_dim;
			if ((rc = check_rows(ctx, q, ldq, w, who, "q")) != NHB_OK || (rc = check_rows(ctx, out, ldo, w, who, "out")) != NHB_OK)
				return rc;
			if (rows_overlap(q, ldq, w, M, out, ldo, w, M))
				return fail(ctx, NHB_ERR_ARG, std::string(who) + ": q and out overlap");
			if (!ctx)
				return fail(ctx, NHB_ERR_ARG, std::string(who) + ": null context");
			device_guard g(ctx->device);
			attn_args a{};
			a.q			   = q;
			a.out		   = out;
			a.ldq		   = ldq;
			a.ldo		   = ldo;
			a.seqs		   = seqs;
			a.cu		   = cu;
			a.n			   = static_cast<int>(n);
			a.heads		   = static_cast<int>(heads);
			a.group		   = a.heads / c.kv_heads;
			a.layer		   = static_cast<int>(layer);
			a.M			   = static_cast<int>(M);
			a.shared_pages = static_cast<int>(shared >> c.page_shift);
			a.scale2	   = scale * 1.4426950408889634f;
			void* ws = nullptr;
			if (cu) {
				if ((rc = wait_pending(ctx)) != NHB_OK)
					return rc;
				return launch_attn_prompt(ctx, c, a);
			}
			// what the batch shares is read once, by its own launch, whose partial results the decode kernel joins.  One sequence
			// shares with nobody.  (Worth its launches for long prefixes only, which is left to the caller.  bf16, up to 700 keys of their own, with
			// the launches / with shared = 0: 64 sequences behind 12288 tokens 106 / 483 us, 1024 74 / 70, 512 74 / 52; 8 behind 12288 49 / 70, 4096 39 / 33.)
			attn_prefix pre{};
			prefix_plan plan{};
			const bool prefix = a.shared_pages > 0 && a.n > 1;
			if (prefix)
				plan = plan_prefix(ctx, c, a);
			const size_t own = (attn_decode_ws_bytes(ctx, c, a) + 255) & ~size_t(255);
			if ((rc = kv_workspace(ctx, own + plan.bytes, &ws, who)) != NHB_OK || (rc = wait_pending(ctx)) != NHB_OK)
				return rc;
			if (prefix && (rc = launch_attn_prefix(ctx, c, a, plan, static_cast<char*>(ws) + own, &pre)) != NHB_OK)
				return rc;
			return launch_attn_decode(ctx, c, a, pre, ws);
		}

	}

}

using namespace nhb;

extern "C" {

int nhb_attn_prompt(nhb_ctx* ctx, const nhb_kv_cache* cache, int64_t layer, const float* q_dev, int64_t ldq, int64_t heads, int64_t M, const int32_t* seqs_dev,
	const int32_t* cu_dev, int64_t n, float scale, float* out_dev, int64_t ldo) {
	if (n > 0 && !cu_dev)
		return fail(ctx, NHB_ERR_ARG, "nhb_attn_prompt: null cu");
	return run_attention(ctx, cache, layer, q_dev, ldq, heads, M, seqs_dev, cu_dev, n, 0, scale, out_dev, ldo, "nhb_attn_prompt");
}

int nhb_attn_decode(nhb_ctx* ctx, const nhb_kv_cache* cache, int64_t layer, const float* q_dev, int64_t ldq, int64_t heads, const int32_t* seqs_dev, int64_t n,
	int64_t shared, float scale, float* out_dev, int64_t ldo) {
	if (shared < 0 || shared > (int64_t(1) << 30))
		return fail(ctx, NHB_ERR_ARG, "nhb_attn_decode: shared is 0 to 2^30 tokens");
	return run_attention(ctx, cache, layer, q_dev, ldq, heads, n, seqs_dev, nullptr, n, shared, scale, out_dev, ldo, "nhb_attn_decode");
}
}
