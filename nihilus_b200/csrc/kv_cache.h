// The paged K/V cache as the kernels see it, the checks its entry points share, and the workspace they use.  Not part of the ABI.
#pragma once
#include "api_types.h"

#define NHB_KV_MAX_SEQS 65536
#define NHB_KV_MAX_PAGES (1 << 24)
#define NHB_KV_COUNTERS 65536
#define NHB_KV_COUNTER_BYTES (NHB_KV_COUNTERS * sizeof(unsigned))

namespace nhb {

	// Status word that a refused nhb_kv_reserve sets beside the first.  Until nhb_sync has reported it, reserve and append change nothing: the
	// last tokens of a sequence are then not those that the caller appends, and storing them would overwrite older ones.
	constexpr int KV_REFUSED = 1;

	// nhb_kv_cache with 32-bit sizes (check_cache has found that they fit)
	struct kv_view {
		char* k;// [n_layers][n_pages][kv_heads][page_tokens][head_dim], 2-byte values
		char* v;
		int32_t* table;// [max_seqs][max_pages]
		int32_t* lens;// [max_seqs]
		int32_t* refs;// [n_pages]
		int n_layers, n_pages, kv_heads, page_tokens, page_shift, head_dim, max_seqs, max_pages;
		int bf16;
		int* status;// the context's device status words (KV_REFUSED: the second)
		long long layer_bytes;// of k and of v
	};

	// tokens a sequence can hold
	__host__ __device__ __forceinline__ int kv_capacity(const kv_view& c) {
		return c.max_pages << c.page_shift;
	}
	__host__ __device__ __forceinline__ int kv_pages_of(const kv_view& c, int tokens) {
		return (tokens + c.page_tokens - 1) >> c.page_shift;
	}

	// (the checks take a null context too, so that they say what is wrong with the other arguments first)
	int check_cache(nhb_ctx* ctx, const nhb_kv_cache* cache, kv_view* out, const char* who);
	int check_layer(nhb_ctx* ctx, const kv_view& c, int64_t layer, const char* who);
	// rows of `width` f32 values: 16-byte aligned, ld a multiple of 4
	int check_rows(nhb_ctx* ctx, const float* p, int64_t ld, int64_t width, const char* who, const char* what);
	int check_list(nhb_ctx* ctx, const int32_t* seqs, const int32_t* cu, int64_t n, const char* who);
	bool rows_overlap(const float* a, int64_t lda, int64_t wa, int64_t ma, const float* b, int64_t ldb, int64_t wb, int64_t mb);

	// One workspace per context for the cache's operators.  Calls follow one another on the context's stream; when the stream changes, the first
	// use on the new one waits for the old one's last.  A buffer that was outgrown is kept until
	// the context ends: a captured graph may still name it.  In front of the bytes handed out lie NHB_KV_COUNTERS arrival counters
	// (kv_counters), zero between launches.
	int kv_workspace(nhb_ctx* ctx, size_t bytes, void** out, const char* who);

	inline unsigned* kv_counters(nhb_ctx* ctx) {
		return static_cast<unsigned*>(ctx->kv_ws);
	}

	// lets a kernel have `bytes` of dynamic shared memory on the context's device: asked once per context
	inline int kv_allow_smem(nhb_ctx* ctx, const void* kern, int bytes) {
		if (std::find(ctx->kv_smem_set.begin(), ctx->kv_smem_set.end(), kern) != ctx->kv_smem_set.end())
			return NHB_OK;
		NHB_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
		ctx->kv_smem_set.push_back(kern);
		return NHB_OK;
	}

	// a launch with the context's programmatic-dependent-launch setting
	template<typename kern_t, typename... args_t> cudaError_t kv_launch(nhb_ctx* ctx, kern_t kern, dim3 grid, dim3 block, size_t smem, args_t... args) {
		cudaLaunchConfig_t lc{};
		lc.gridDim			= grid;
		lc.blockDim			= block;
		lc.dynamicSmemBytes = smem;
		lc.stream			= ctx->stream;
		cudaLaunchAttribute attr[1];
		attr[0].id										   = cudaLaunchAttributeProgrammaticStreamSerialization;
		attr[0].val.programmaticStreamSerializationAllowed = 1;
		lc.attrs										   = attr;
		lc.numAttrs										   = ctx->pdl ? 1 : 0;
		cudaError_t e = cudaLaunchKernelEx(&lc, kern, args...);
		if (e == cudaSuccess)
			ctx->launches += 1;
		return e;
	}

}
