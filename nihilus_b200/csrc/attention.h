// What the two attention kernels (attn_prompt.cu, attn_decode.cu) share: arguments, tensor maps of the pages, the split of f32 into
// two 16-bit parts.  Not part of the ABI.
#pragma once
#include <cuda_bf16.h>

#include "kv_cache.h"
#include "tc_ptx.cuh"

namespace nhb {

	struct attn_args {
		const float* q;
		float* out;
		long long ldq, ldo;
		const int *seqs, *cu;
		int n;// list entries
		int heads, group;// query heads, and those on one kv head
		int layer;
		int M;// rows
		int shared_pages;// decode: whole pages that all entries have in common
		float scale2;// scale * log2(e): scores are kept in powers of two
	};

	// Partial results of the keys that a batch shares (attn_prompt.cu), joined with each sequence's own keys by the decode kernel: per kv head
	// the unnormalised outputs and (maximum, sum) of every row, row = list entry * group + head of the group
	struct attn_prefix {
		const float* o;// [kv_heads][stride][head_dim], the first `rows` of each kv head
		const float2* ml;// [kv_heads][stride]
		long long stride;// rows of a kv head: the other splits' parts, joined into the first, lie behind
		int any;// 0: nothing shared
	};

	// One layer's k or v as rows of head_dim: a box is 64 columns (128 bytes, the swizzle's span) by a page's rows
	inline bool make_page_map(CUtensorMap* map, const kv_view& c, const char* pool, int layer) {
		tensor_map_encode_t fn = tensor_map_encode();
		if (!fn)
			return false;
		const cuuint64_t dims[2]	= { static_cast<cuuint64_t>(c.head_dim), static_cast<cuuint64_t>(c.n_pages) * c.kv_heads * c.page_tokens };
		const cuuint64_t strides[1] = { static_cast<cuuint64_t>(c.head_dim) * 2 };
		const cuuint32_t box[2]		= { 64, static_cast<cuuint32_t>(c.page_tokens < 64 ? c.page_tokens : 64) };
		const cuuint32_t estr[2]	= { 1, 1 };
		void* base					= const_cast<char*>(pool) + static_cast<size_t>(layer) * c.layer_bytes;
		return fn(map, c.bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
				   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
	}

	// attn_decode.cu
	int launch_attn_decode(nhb_ctx* ctx, const kv_view& c, const attn_args& a, const attn_prefix& pre, void* ws);
	size_t attn_decode_ws_bytes(const nhb_ctx* ctx, const kv_view& c, const attn_args& a);

	// attn_prompt.cu
	int launch_attn_prompt(nhb_ctx* ctx, const kv_view& c, const attn_args& a);
	struct prefix_plan {
		bool two;// two row tiles per CTA
		long long row_tiles;
		int splits, tiles_per_split;
		size_t bytes;// of workspace
	};
	prefix_plan plan_prefix(const nhb_ctx* ctx, const kv_view& c, const attn_args& a);
	int launch_attn_prefix(nhb_ctx* ctx, const kv_view& c, const attn_args& a, const prefix_plan& plan, void* ws, attn_prefix* out);

	// ---- device helpers ----
	__device__ __forceinline__ float ex2(float x) {
		float y;
		asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
		return y;
	}

	// (a, b) as 16-bit pairs hi + lo: hi rounds to nearest, lo rounds what is left, so the pair is off by at most 2^-22 (f16) or
	// 2^-16 (bf16) of its value.  hi infinite or NaN: lo is NaN, and so is whatever it enters.
	template<bool BF16> __device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
		if constexpr (BF16) {
			const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
			const __nv_bfloat162 l = __floats2bfloat162_rn(a - __low2float(h), b - __high2float(h));
			hi = *reinterpret_cast<const uint32_t*>(&h);
			lo = *reinterpret_cast<const uint32_t*>(&l);
		} else {
			const __half2 h = __floats2half2_rn(a, b);
			const __half2 l = __floats2half2_rn(a - __low2float(h), b - __high2float(h));
			hi = *reinterpret_cast<const uint32_t*>(&h);
			lo = *reinterpret_cast<const uint32_t*>(&l);
		}
	}

	// The largest weight of a tile is 2 to this.  f16: 2^14, so that small weights keep all their parts normal numbers; bf16, with f32's range, 1, so
	// that sums of weights times values stay in range where f32's do.  (Outputs are divided by the sum of the weights.)
	template<bool BF16> constexpr float WEIGHT_BITS = BF16 ? 0.f : 14.f;

	// A row of queries is scaled by a power of two that brings its largest element to [2^12, 2^13) before it is split for f16: both 16-bit
	// parts are then normal numbers for all elements that matter, whatever the row's size.  Returns the factor; *back undoes it.
	// bf16 has f32's range: its rows are split as they are, so that their products with keys of any size stay in range where f32's do.
	__device__ __forceinline__ float row_scaling(float amax, float* back) {
		int e = static_cast<int>((__float_as_uint(amax) >> 23) & 255u) - 127 - 12;
		if (amax == 0.f || e > 115)// zero, or infinite / NaN / next to the largest f32
			e = amax == 0.f ? 0 : 115;
		e	  = max(e, -100);
		*back = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
		return __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
	}

}
