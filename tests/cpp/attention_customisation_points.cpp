// Must compile: the customisation points of mega_dispatch.hpp for rope + cache write and for attention as calls of attention_abi.h, for a config that
// does not ask for the stand-ins.  The test suite compiles this file with -fsyntax-only.
#include <nihilus_amd/attention_abi.h>
#include <nihilus_amd/mega_dispatch.hpp>

#define mock_config my_config // the mock graph, under a config name of its own
#define amd_matmul_only stand_ins_are_allowed // ... that asks for none
#include "mock_model.hpp"
#undef amd_matmul_only
#undef mock_config

#include <cmath>

namespace {
	using mtt = nihilus::tiny_llama_traits;
	constexpr int64_t q_heads = mtt::attention_head_count, embedding = mtt::embedding_length, kv_width = mtt::n_embd_kv_gqa, head_dim = mtt::rope_dimension_count;

	// one layer's pages, the batch's tables, the turns of rope_freqs, workspaces and zeroed counters: the host's, on the device
	nh_attn_cache caches[mtt::block_count]{};
	nh_attn_batch my_batch{};
	const double* turns{};
	void *workspace{}, *counters{};
	int64_t workspace_bytes{}, counter_bytes{};

	nh_attn_cache my_cache(int64_t block) {
		return caches[block];
	}
	void my_check(int status) {
		nihilus::amd_detail::check<nihilus::my_config>(status, "attention");
	}
}

template<> struct nihilus::amd_qkv_epilogue<nihilus::my_config> {
	template<typename core> static void impl(core&, int64_t block, uint64_t rows, float* q, const float* k, const float* v, void* stream) {
		const nh_attn_cache cache = my_cache(block);
		my_check(nh_attn_append_rope(&cache, &my_batch, q, k, v, q, NH_F32, static_cast<int64_t>(rows), q_heads, embedding, kv_width, kv_width, turns, head_dim / 2, 1, stream));
	}
};
template<> struct nihilus::amd_attention<nihilus::my_config> {
	template<typename core> static const float* impl(core& params, int64_t block, uint64_t rows, float* scratch, void* stream) {
		const float* q			  = params.data_ptrs.template get_q_input_data<float>();
		const nh_attn_cache cache = my_cache(block);
		const float scale		  = 1.0f / std::sqrt(static_cast<float>(head_dim));
		if (my_batch.starts) {
			my_check(nh_attn_prompt(&cache, &my_batch, q, scratch, NH_F32, static_cast<int64_t>(rows), q_heads, embedding, scale, workspace, workspace_bytes, counters, counter_bytes, stream));
		} else {
			my_check(nh_attn_decode(&cache, &my_batch, nullptr, 0, q, scratch, NH_F32, q_heads, embedding, scale, workspace, workspace_bytes, counters, counter_bytes, stream));
		}
		return scratch;
	}
};

using namespace nihilus;
using qkv_core	= core_traits_old<my_config, core_types::mega_qkv_prep_and_cache_publish>;
using attn_core = core_traits_old<my_config, core_types::mega_attention_apply>;

void instantiate(qkv_core& qkv, attn_core& attn) {
	kernel_dispatcher_impl<my_config, qkv_core, device_types::gpu, gfx950_arch_index, core_types::mega_qkv_prep_and_cache_publish, processing_phases::prompt_eval_time>::impl(qkv, 0);
	kernel_dispatcher_impl<my_config, qkv_core, device_types::gpu, gfx950_arch_index, core_types::mega_qkv_prep_and_cache_publish, processing_phases::eval_time>::impl(qkv, 0);
	kernel_dispatcher_impl<my_config, attn_core, device_types::gpu, gfx950_arch_index, core_types::mega_attention_apply, processing_phases::prompt_eval_time>::impl(attn, 0);
	kernel_dispatcher_impl<my_config, attn_core, device_types::gpu, gfx950_arch_index, core_types::mega_attention_apply, processing_phases::eval_time>::impl(attn, 0);
}
