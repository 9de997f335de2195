// extern "C" surface of the attention and cache calls: argument checks, then the launch functions.  What lies in device memory (tables,
// lengths, starts) cannot be looked at here; the kernels check it where they use it.
#include "../../include/nihilus_amd/attention_abi.h"
#include "abi_checks.h"
#include "attention_device.h"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdlib>
#include <iterator>

namespace {

using nh::aligned16;
using nh::as_stream;
using nh::from_hip;
using nh::overlap;
using nh::require_device;

// row, token and tile numbers are 32-bit inside the kernels, with room for sums of two
constexpr int64_t MAX_KEYS		= int64_t{ 1 } << 30; // of a sequence's table, of a prefix
constexpr int64_t MAX_ROW_HEADS = int64_t{ 1 } << 30; // rows * q_heads
constexpr int64_t MAX_SEQUENCES = int64_t{ 1 } << 20;
constexpr int64_t MAX_ALL_KEYS	= int64_t{ 1 } << 35; // sequences * keys of a table: their number in steps of 32 is a 32-bit sum

inline int page_shift(int64_t page_size) {
	for (int shift = 4; shift <= 8; ++shift) {
		if (page_size == int64_t{ 1 } << shift) {
			return shift;
		}
	}
	return -1;
}
inline int check_cache(const nh_attn_cache* c) {
	NH_REQUIRE(c, NH_ERR_NULL_POINTER);
	NH_REQUIRE(c->type == NH_F16 || c->type == NH_BF16, NH_ERR_ARGUMENT);
	NH_REQUIRE(c->layers > 0 && c->pages > 0 && c->kv_heads > 0 && page_shift(c->page_size) > 0 && (c->head_dim == 64 || c->head_dim == 128), NH_ERR_SHAPE);
	NH_REQUIRE(c->layers <= 65536 && c->kv_heads < 65536 && c->pages <= (int64_t{ 1 } << 28), NH_ERR_TOO_LARGE);
	NH_REQUIRE(c->k_pages && c->v_pages, NH_ERR_NULL_POINTER);
	NH_REQUIRE(aligned16(c->k_pages) && aligned16(c->v_pages), NH_ERR_ALIGNMENT);
	return NH_OK;
}
// for batches that have sequences
inline int check_batch(const nh_attn_batch* b, int64_t page_size) {
	NH_REQUIRE(b, NH_ERR_NULL_POINTER);
	NH_REQUIRE(b->sequences >= 0 && b->table_width >= 0, NH_ERR_SHAPE);
	NH_REQUIRE(b->sequences <= MAX_SEQUENCES && b->table_width <= MAX_KEYS / page_size && b->sequences * b->table_width * page_size <= MAX_ALL_KEYS, NH_ERR_TOO_LARGE);
	NH_REQUIRE(b->sequences == 0 || (b->lengths && (b->page_table || b->table_width == 0)), NH_ERR_NULL_POINTER);
	return NH_OK;
}
inline int64_t value_bytes(int type) {
	return type == NH_F32 ? 4 : 2;
}
// q (k, v, out): type, heads, strides
inline int check_rows(const nh_attn_cache* c, int type, int64_t rows, int64_t heads, int64_t stride) {
	NH_REQUIRE(type == NH_F32 || type == c->type, NH_ERR_ARGUMENT);
	NH_REQUIRE(rows >= 0 && heads > 0 && heads % c->kv_heads == 0, NH_ERR_SHAPE);
	NH_REQUIRE(heads < 65536 && rows <= MAX_ROW_HEADS / heads, NH_ERR_TOO_LARGE);
	NH_REQUIRE(stride >= heads * c->head_dim && stride <= (int64_t{ 1 } << 40), NH_ERR_SHAPE);
	NH_REQUIRE(stride * value_bytes(type) % 16 == 0, NH_ERR_ALIGNMENT);
	return NH_OK;
}
// bytes that rows of a stride reach over
inline int64_t span(int64_t rows, int64_t heads, int64_t head_dim, int64_t stride, int type) {
	return ((rows - 1) * stride + heads * head_dim) * value_bytes(type);
}
inline nh::cache_view view(const nh_attn_cache* c) {
	return nh::cache_view{ static_cast<uint16_t*>(c->k_pages), static_cast<uint16_t*>(c->v_pages), c->kv_heads * c->page_size * c->head_dim, static_cast<int>(c->pages),
		static_cast<int>(c->kv_heads), page_shift(c->page_size) };
}
inline nh::batch_view view(const nh_attn_batch* b) {
	return nh::batch_view{ b->page_table, b->lengths, b->starts, static_cast<int>(b->sequences), static_cast<int>(b->table_width) };
}

std::atomic<int> forced_prompt_kernel{ 0 };

} // namespace

// Whether a decode step's shared prefix is gone over once for all sequences, by the tile kernel, or by each with its own keys.  The first takes a launch more
// and the join of its results, some 7 us and more with more sequences; the second reads the prefix from the caches once for each sequence.
// us, apart | with their own (fp16, own keys 200; 32 / 8 heads of 128): prefix 1024: 8 sequences 16.3 | 12.3, 64 28.6 | 25.0;  4096: 8 19.9 | 16.9, 16 24.3 | 27.1,
// 64 35.1 | 61.2;  8192: 4 23.6 | 17.2, 8 24.4 | 25.3, 16 27.0 | 42.2;  16 / 2 heads, 8192: 32 34.2 | 27.3, 64 30.5 | 42.0
static bool prefix_apart(int64_t sequences, int64_t kv_heads, int64_t head_dim, int64_t prefix_keys) {
	if (const int forced = forced_prompt_kernel.load(std::memory_order_relaxed)) {
		return forced == 2;
	}
	return static_cast<double>(sequences) * static_cast<double>(kv_heads * head_dim) * static_cast<double>(prefix_keys) > 67108864.0;
}

bool nh::prompt_by_rows(int64_t rows, int64_t sequences, int64_t q_heads, int64_t kv_heads) {
	if (const int forced = forced_prompt_kernel.load(std::memory_order_relaxed)) {
		return forced == 1;
	}
	if (sequences <= 0 || kv_heads <= 0) {
		return true;
	}
	// The rows kernel reads a sequence's keys again for every 16 rows, but spreads any shape over the chip; the tile kernel reads them for every 128, and a
	// workgroup's way to its first result is longer.  So: the first while its row groups are all on the chip at once, or where no tile has more than one.
	// us, rows | tiles (fp16, 32 / 8 heads of 128 where nothing else is said):
	//   256 row groups:  a prompt of 128 rows 7.0 | 12.8, behind 1024 keys 18 | 23, behind 8192 keys 68 | 40
	//   512:             a prompt of 256 rows 8.7 | 14.3, behind 1024 keys 23 | 24, behind 8192 keys 120 | 55; 8 of 32 rows 6.8 | 11.6
	//   1024:            a prompt of 512 rows 20.0 | 18.5, behind 1024 keys 44 | 28, behind 8192 keys 231 | 91; 16 / 2 heads of 64, 64 of 16 rows 8.7 | 8.4
	//   2048:            8 prompts of 128 rows 21 | 15, 64 of 16 rows 19 | 11.5; but 32 / 32 heads, 64 of 16 rows, each tile with one row group: 21 | 34
	// (How many keys there are is not known on the host: a table has room for more.)
	const int64_t each = (rows + sequences - 1) / sequences * (q_heads / kv_heads); // the lengths are not known here: as if all were alike
	const int64_t row_groups = sequences * kv_heads * ((each + 15) / 16), tiles = sequences * kv_heads * ((each + 127) / 128);
	return row_groups <= 512 || row_groups <= tiles;
}

extern "C" {

int nh_attn_append_rope(const nh_attn_cache* host_cache, const nh_attn_batch* host_batch, const void* q, const void* k, const void* v, void* q_out, int type, int64_t rows, int64_t q_heads,
	int64_t q_stride, int64_t k_stride, int64_t v_stride, const double* turns, int64_t pairs, int interleaved, void* stream) {
	NH_TRY(check_cache(host_cache));
	NH_REQUIRE(host_cache->layers == 1, NH_ERR_SHAPE);
	NH_TRY(check_batch(host_batch, host_cache->page_size));
	NH_TRY(check_rows(host_cache, type, rows, q_heads, q_stride));
	NH_TRY(check_rows(host_cache, type, rows, host_cache->kv_heads, k_stride));
	NH_TRY(check_rows(host_cache, type, rows, host_cache->kv_heads, v_stride));
	NH_REQUIRE(pairs >= 0 && pairs % 8 == 0 && 2 * pairs <= host_cache->head_dim, NH_ERR_SHAPE);
	NH_REQUIRE(host_batch->starts || rows == host_batch->sequences, NH_ERR_ARGUMENT);
	NH_REQUIRE(nh::append_rope_fits(rows, host_cache->kv_heads), NH_ERR_TOO_LARGE);
	if (rows == 0 || host_batch->sequences == 0) {
		return NH_OK;
	}
	NH_REQUIRE(q && k && v && q_out && (turns || pairs == 0), NH_ERR_NULL_POINTER);
	NH_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(q_out), NH_ERR_ALIGNMENT);
	const int64_t dim = host_cache->head_dim, kv_heads = host_cache->kv_heads, out_bytes = span(rows, q_heads, dim, q_heads * dim, type);
	NH_REQUIRE(q_out == q ? q_stride == q_heads * dim : !overlap(q_out, out_bytes, q, span(rows, q_heads, dim, q_stride, type)), NH_ERR_ARGUMENT);
	NH_REQUIRE(!overlap(q_out, out_bytes, k, span(rows, kv_heads, dim, k_stride, type)) && !overlap(q_out, out_bytes, v, span(rows, kv_heads, dim, v_stride, type)), NH_ERR_ARGUMENT);
	NH_TRY(require_device());
	nh::append_args a{};
	a.cache = view(host_cache), a.batch = view(host_batch);
	a.q = q, a.k = k, a.v = v, a.q_out = q_out, a.turns = turns;
	a.q_stride = q_stride, a.k_stride = k_stride, a.v_stride = v_stride;
	a.rows = static_cast<int>(rows), a.q_heads = static_cast<int>(q_heads), a.head_dim = static_cast<int>(host_cache->head_dim), a.pairs = static_cast<int>(pairs);
	a.interleaved = interleaved != 0;
	return from_hip(nh::launch_append_rope(a, host_cache->type, type, as_stream(stream)));
}

static int check_attention(const nh_attn_cache* c, const nh_attn_batch* b, int type, int64_t rows, int64_t q_heads, int64_t q_stride, float scale) {
	NH_TRY(check_cache(c));
	NH_REQUIRE(c->layers == 1, NH_ERR_SHAPE);
	NH_TRY(check_batch(b, c->page_size));
	NH_TRY(check_rows(c, type, rows, q_heads, q_stride));
	NH_REQUIRE(scale > 0.0f && std::isfinite(scale), NH_ERR_ARGUMENT);
	return NH_OK;
}
static nh::attention_args attention(const nh_attn_cache* c, const nh_attn_batch* b, const void* q, void* out, int64_t rows, int64_t q_heads, int64_t q_stride, float scale) {
	nh::attention_args a{};
	a.cache = view(c), a.batch = view(b);
	a.q = q, a.out = out, a.q_stride = q_stride;
	a.rows = static_cast<int>(rows), a.q_heads = static_cast<int>(q_heads), a.head_dim = static_cast<int>(c->head_dim);
	a.scale = scale;
	return a;
}

static bool out_over_q(const nh_attn_cache* c, const void* q, const void* out, int type, int64_t rows, int64_t q_heads, int64_t q_stride) {
	return overlap(out, span(rows, q_heads, c->head_dim, q_heads * c->head_dim, type), q, span(rows, q_heads, c->head_dim, q_stride, type));
}

static int check_memory(int64_t workspace_need, int64_t counter_need, const void* workspace, int64_t workspace_bytes, const void* counters, int64_t counter_bytes) {
	NH_REQUIRE((workspace || workspace_need == 0) && (counters || counter_need == 0), NH_ERR_NULL_POINTER);
	NH_REQUIRE(((reinterpret_cast<uintptr_t>(workspace) | reinterpret_cast<uintptr_t>(counters)) & 255u) == 0, NH_ERR_ALIGNMENT);
	NH_REQUIRE(workspace_bytes >= workspace_need && counter_bytes >= counter_need, NH_ERR_ARGUMENT);
	return NH_OK;
}
static int check_heads(int64_t rows, int64_t sequences, int64_t q_heads, int64_t kv_heads, int64_t head_dim, const int64_t* a, const int64_t* b) {
	NH_REQUIRE(a && b, NH_ERR_NULL_POINTER);
	NH_REQUIRE(rows >= 0 && sequences >= 0 && q_heads > 0 && kv_heads > 0 && q_heads % kv_heads == 0 && (head_dim == 64 || head_dim == 128), NH_ERR_SHAPE);
	NH_REQUIRE(sequences <= MAX_SEQUENCES && q_heads < 65536 && rows <= MAX_ROW_HEADS / q_heads && sequences * kv_heads <= MAX_ROW_HEADS / 4, NH_ERR_TOO_LARGE);
	return NH_OK;
}

int nh_attn_prompt_needs(int64_t rows, int64_t sequences, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t* host_workspace_bytes, int64_t* host_counter_bytes) {
	NH_TRY(check_heads(rows, sequences, q_heads, kv_heads, head_dim, host_workspace_bytes, host_counter_bytes));
	const bool by_rows = nh::prompt_by_rows(rows, sequences, q_heads, kv_heads);
	NH_REQUIRE(by_rows || nh::attention_tiles_fit(rows, sequences, q_heads, kv_heads), NH_ERR_TOO_LARGE);
	const nh::attention_needs n = rows == 0 || sequences == 0 ? nh::attention_needs{ 0, 0 }
		: by_rows												  ? nh::attention_rows_needs(sequences, false, q_heads, kv_heads, head_dim, 0)
																  : nh::attention_tiles_needs(rows, sequences, q_heads, kv_heads, head_dim);
	*host_workspace_bytes		= n.workspace;
	*host_counter_bytes			= n.counters;
	return NH_OK;
}

int nh_attn_prompt(const nh_attn_cache* host_cache, const nh_attn_batch* host_batch, const void* q, void* out, int type, int64_t rows, int64_t q_heads, int64_t q_stride, float scale,
	void* workspace, int64_t workspace_bytes, void* counters, int64_t counter_bytes, void* stream) {
	NH_TRY(check_attention(host_cache, host_batch, type, rows, q_heads, q_stride, scale));
	int64_t need = 0, counter_need = 0;
	NH_TRY(nh_attn_prompt_needs(rows, host_batch->sequences, q_heads, host_cache->kv_heads, host_cache->head_dim, &need, &counter_need));
	if (rows == 0 || host_batch->sequences == 0) {
		return NH_OK;
	}
	NH_REQUIRE(host_batch->starts && q && out, NH_ERR_NULL_POINTER);
	NH_REQUIRE(aligned16(q) && aligned16(out), NH_ERR_ALIGNMENT);
	NH_REQUIRE(!out_over_q(host_cache, q, out, type, rows, q_heads, q_stride), NH_ERR_ARGUMENT);
	NH_TRY(check_memory(need, counter_need, workspace, workspace_bytes, counters, counter_bytes));
	NH_TRY(require_device());
	nh::attention_args a = attention(host_cache, host_batch, q, out, rows, q_heads, q_stride, scale);
	a.workspace			 = workspace;
	a.counters			 = static_cast<int32_t*>(counters);
	bool by_rows		 = nh::prompt_by_rows(rows, host_batch->sequences, q_heads, host_cache->kv_heads);
	if (by_rows && !nh::attention_rows_fit(rows, host_batch->sequences, false, q_heads / host_cache->kv_heads, host_batch->table_width * host_cache->page_size)) {
		NH_REQUIRE(nh::attention_tiles_fit(rows, host_batch->sequences, q_heads, host_cache->kv_heads), NH_ERR_TOO_LARGE);
		by_rows		= false; // few rows against tables of a billion keys: more work than the rows kernel can number; the tile kernel without memory of its own
		a.workspace = nullptr;
	}
	return from_hip(by_rows ? nh::launch_attention_rows(a, host_cache->type, type, as_stream(stream)) : nh::launch_attention_tiles(a, host_cache->type, type, as_stream(stream)));
}

int nh_attn_debug_prompt_kernel(int64_t rows, int64_t sequences, int64_t q_heads, int64_t kv_heads, int force) {
	if (force != -1) {
		const char* hooks = std::getenv("NH_Q8_0_DEBUG_HOOKS");
		NH_REQUIRE(hooks && hooks[0] == '1' && hooks[1] == '\0' && force >= 0 && force <= 2, NH_ERR_ARGUMENT);
		forced_prompt_kernel.store(force, std::memory_order_relaxed);
	}
	return nh::prompt_by_rows(rows, sequences, q_heads, kv_heads) ? 1 : 2;
}

int nh_attn_decode_needs(int64_t sequences, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t prefix_count, int64_t page_size, int64_t* host_workspace_bytes,
	int64_t* host_counter_bytes) {
	NH_TRY(check_heads(sequences, sequences, q_heads, kv_heads, head_dim, host_workspace_bytes, host_counter_bytes));
	NH_REQUIRE(prefix_count >= 0 && page_shift(page_size) > 0, NH_ERR_SHAPE);
	NH_REQUIRE(prefix_count <= MAX_KEYS / page_size, NH_ERR_TOO_LARGE);
	NH_REQUIRE(nh::prefix_fits(nh::plan_prefix(sequences, q_heads / kv_heads, kv_heads, prefix_count * page_size), kv_heads), NH_ERR_TOO_LARGE);
	const nh::attention_needs n = nh::attention_rows_needs(sequences, true, q_heads, kv_heads, head_dim, prefix_count * page_size);
	*host_workspace_bytes		= n.workspace;
	*host_counter_bytes			= n.counters;
	return NH_OK;
}

int nh_attn_decode(const nh_attn_cache* host_cache, const nh_attn_batch* host_batch, const int32_t* prefix_pages, int64_t prefix_count, const void* q, void* out, int type, int64_t q_heads,
	int64_t q_stride, float scale, void* workspace, int64_t workspace_bytes, void* counters, int64_t counter_bytes, void* stream) {
	NH_REQUIRE(host_batch, NH_ERR_NULL_POINTER);
	NH_TRY(check_attention(host_cache, host_batch, type, host_batch->sequences, q_heads, q_stride, scale));
	NH_REQUIRE(!host_batch->starts, NH_ERR_ARGUMENT);
	NH_REQUIRE(nh::attention_rows_fit(host_batch->sequences, host_batch->sequences, true, q_heads / host_cache->kv_heads, host_batch->table_width * host_cache->page_size), NH_ERR_TOO_LARGE);
	int64_t need = 0, counter_need = 0;
	NH_TRY(nh_attn_decode_needs(host_batch->sequences, q_heads, host_cache->kv_heads, host_cache->head_dim, prefix_count, host_cache->page_size, &need, &counter_need));
	if (host_batch->sequences == 0) {
		return NH_OK;
	}
	NH_REQUIRE(q && out && (prefix_pages || prefix_count == 0), NH_ERR_NULL_POINTER);
	NH_REQUIRE(aligned16(q) && aligned16(out), NH_ERR_ALIGNMENT);
	NH_REQUIRE(!out_over_q(host_cache, q, out, type, host_batch->sequences, q_heads, q_stride), NH_ERR_ARGUMENT);
	NH_TRY(check_memory(need, counter_need, workspace, workspace_bytes, counters, counter_bytes));
	NH_TRY(require_device());
	nh::attention_args a = attention(host_cache, host_batch, q, out, host_batch->sequences, q_heads, q_stride, scale);
	a.prefix_pages		 = prefix_pages;
	a.prefix_count		 = static_cast<int>(prefix_count);
	a.prefix_apart		 = prefix_count > host_batch->table_width || prefix_apart(host_batch->sequences, host_cache->kv_heads, host_cache->head_dim, prefix_count * host_cache->page_size);
	a.workspace			 = workspace;
	a.counters			 = static_cast<int32_t*>(counters);
	return from_hip(nh::launch_attention_rows(a, host_cache->type, type, as_stream(stream)));
}

int64_t nh_attn_pages_workspace_bytes(int64_t pages, int64_t sequences, int64_t table_width) {
	if (pages <= 0 || sequences < 0 || table_width < 0) {
		return NH_ERR_SHAPE;
	}
	if (pages > (int64_t{ 1 } << 28) || sequences > MAX_SEQUENCES) {
		return NH_ERR_TOO_LARGE;
	}
	return nh::cache_pages_workspace(pages, sequences, table_width);
}

static int check_pages(const nh_attn_cache* c, const nh_attn_batch* b, int64_t children, const int32_t* new_table, const int32_t* info, const void* workspace, int64_t workspace_bytes) {
	NH_TRY(check_cache(c));
	NH_TRY(check_batch(b, c->page_size));
	NH_REQUIRE(children >= 0, NH_ERR_SHAPE);
	// (the page calls count a table's entries in 32 bits)
	NH_REQUIRE(children <= MAX_SEQUENCES && children * b->table_width * c->page_size <= MAX_ALL_KEYS && children * b->table_width <= INT32_MAX, NH_ERR_TOO_LARGE);
	const int64_t need = nh_attn_pages_workspace_bytes(c->pages, children, b->table_width);
	NH_REQUIRE(need >= 0, static_cast<int>(need));
	NH_REQUIRE(info && (workspace || need == 0) && (new_table || children * b->table_width == 0), NH_ERR_NULL_POINTER);
	NH_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 255u) == 0, NH_ERR_ALIGNMENT);
	NH_REQUIRE(workspace_bytes >= need, NH_ERR_ARGUMENT);
	return NH_OK;
}
// Nothing that a call on the pages writes may lie over what it reads (every workgroup plans from the inputs while the first one writes the results), nor over
// another result, nor the workspace over either.
static int check_page_results(const nh_attn_cache* c, const nh_attn_batch* b, int64_t children, const int32_t* parents, const int32_t* grow, const int32_t* new_table, const int32_t* new_lengths,
	const int32_t* info, const void* workspace) {
	struct part {
		const void* at;
		int64_t bytes;
	};
	const int64_t cache_bytes = static_cast<int64_t>(
		std::min<__int128>(static_cast<__int128>(c->layers * c->pages) * (c->kv_heads * c->page_size * c->head_dim * 2), int64_t{ 1 } << 62));
	const int64_t need = nh_attn_pages_workspace_bytes(c->pages, children, b->table_width);
	const part inputs[] = { { c->k_pages, cache_bytes }, { c->v_pages, cache_bytes }, { b->page_table, b->sequences * b->table_width * 4 }, { b->lengths, b->sequences * 4 }, { parents, children * 4 },
		{ grow, children * 4 } };
	const part results[] = { { new_table, children * b->table_width * 4 }, { new_lengths, children * 4 }, { info, 12 }, { workspace, need } };
	auto apart = [](const part& x, const part& y) {
		return x.bytes == 0 || y.bytes == 0 || !overlap(x.at, x.bytes, y.at, y.bytes);
	};
	for (const part* r = std::begin(results); r != std::end(results); ++r) {
		for (const part& in : inputs) {
			NH_REQUIRE(apart(*r, in), NH_ERR_ARGUMENT);
		}
		for (const part* other = std::begin(results); other != r; ++other) {
			NH_REQUIRE(apart(*r, *other), NH_ERR_ARGUMENT);
		}
	}
	return NH_OK;
}
static nh::pages_args pages(const nh_attn_cache* c, const nh_attn_batch* b, int32_t* new_table, int32_t* info, void* workspace) {
	nh::pages_args a{};
	a.k = static_cast<uint16_t*>(c->k_pages), a.v = static_cast<uint16_t*>(c->v_pages);
	a.page_bytes = c->kv_heads * c->page_size * c->head_dim * 2;
	a.layers	 = c->layers;
	a.pages		 = static_cast<int>(c->pages);
	a.page_shift = page_shift(c->page_size);
	a.batch		 = view(b);
	a.new_table = new_table, a.info = info, a.workspace = workspace;
	return a;
}

int nh_attn_cache_step(const nh_attn_cache* host_cache, const nh_attn_batch* host_batch, const int32_t* parents, const int32_t* grow, int64_t children, int32_t* new_table, int32_t* new_lengths,
	int32_t* info, void* workspace, int64_t workspace_bytes, void* stream) {
	NH_TRY(check_pages(host_cache, host_batch, children, new_table, info, workspace, workspace_bytes));
	NH_REQUIRE(children == 0 || (parents && grow && new_lengths), NH_ERR_NULL_POINTER);
	NH_TRY(check_page_results(host_cache, host_batch, children, parents, grow, new_table, new_lengths, info, workspace));
	NH_TRY(require_device());
	nh::pages_args a = pages(host_cache, host_batch, new_table, info, workspace);
	a.parents = parents, a.grow = grow, a.new_lengths = new_lengths;
	a.children = static_cast<int>(children);
	return from_hip(nh::launch_cache_step(a, as_stream(stream)));
}

int nh_attn_cache_compact(const nh_attn_cache* host_cache, const nh_attn_batch* host_batch, int32_t* new_table, int32_t* info, void* workspace, int64_t workspace_bytes, void* stream) {
	NH_REQUIRE(host_batch, NH_ERR_NULL_POINTER);
	NH_TRY(check_pages(host_cache, host_batch, host_batch->sequences, new_table, info, workspace, workspace_bytes));
	NH_TRY(check_page_results(host_cache, host_batch, host_batch->sequences, nullptr, nullptr, new_table, nullptr, info, workspace));
	NH_TRY(require_device());
	return from_hip(nh::launch_cache_compact(pages(host_cache, host_batch, new_table, info, workspace), as_stream(stream)));
}

} // extern "C"
