// Device-side helpers shared by the gfx950 attention kernels: operand types of the 16-bit matrix instructions, the paged cache's
// addressing, the splitting of fp32 values into 16-bit terms, and the launch functions each translation unit exports.
#pragma once

#include "../../include/nihilus_amd/attention_abi.h"
#include "q8_0_device.h"

namespace nh {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef unsigned v4u __attribute__((ext_vector_type(4)));

// The matrix instructions of one 16-bit type.  A: 16 (32) rows, B: 16 (32) columns; lane l holds 8 values of row / column l % 16 (32) along the
// axis that is added up, from 8 * (l / 16 (32)) on.  Result: column l % 16 (32); rows 4 (l / 16) + i, or 8 (i / 4) + 4 (l / 32) + i % 4.
template<int TYPE> struct half_type;
template<> struct half_type<NH_F16> {
	using value = _Float16;
	using vec	= v8h;
	static constexpr int terms_of_f32 = 2; // 11 + 11 bits
	static __device__ __forceinline__ v4f mfma16(vec a, vec b, v4f c) {
		return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
	}
	static __device__ __forceinline__ v16f mfma32(vec a, vec b, v16f c) {
		return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
	}
};
template<> struct half_type<NH_BF16> {
	using value = __bf16;
	using vec	= v8b;
	static constexpr int terms_of_f32 = 3; // 8 + 8 + 8 bits
	static __device__ __forceinline__ v4f mfma16(vec a, vec b, v4f c) {
		return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
	}
	static __device__ __forceinline__ v16f mfma32(vec a, vec b, v16f c) {
		return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
	}
};
// fp32 q: as many terms as make up an fp32 value; q of the cache's type: itself
template<int CACHE, int Q> constexpr int terms = Q == NH_F32 ? half_type<CACHE>::terms_of_f32 : 1;

// x as a sum of N values of 16 bits, each the rounded rest of those before it (round to nearest even).  Eight at once, as one operand of
// a matrix instruction for each term.
template<int CACHE, int N> __device__ __forceinline__ void split8(const float (&x)[8], typename half_type<CACHE>::vec (&t)[N]) {
	using value = typename half_type<CACHE>::value;
#pragma unroll
	for (int j = 0; j < 8; ++j) {
		float rest = x[j];
#pragma unroll
		for (int n = 0; n < N; ++n) {
			const value v = static_cast<value>(rest);
			t[n][j]		  = v;
			rest		  = __fsub_rn(rest, static_cast<float>(v));
		}
	}
}

__device__ __forceinline__ float exp2_fast(float x) {
	return __builtin_amdgcn_exp2f(x); // v_exp_f32: 1 ulp; arguments here are below 16 (see weight_bias), results below 2^-126 are flushed, far under a sum that holds a 1
}
// What the sums of a part of the keys are multiplied with when parts are joined: 2^x, x how far (in powers of two) the part's maximum lies below the joint one.
// Never zero: an infinite value has been added to its part by then and has to stay one (infinity times zero is NaN), and 2^-126 of a part shows nowhere
// beside one whose weights add up to 1 and more.
__device__ __forceinline__ float part_factor(float x) {
	return fmaxf(exp2_fast(x), 0x1p-126f);
}
// the value of lane ^ 32 (^ 16)
__device__ __forceinline__ float swap32(float x, int lane) {
	const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
	return __builtin_bit_cast(float, (lane & 32) ? r[0] : r[1]);
}
__device__ __forceinline__ float swap16(float x, int lane) {
	const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
	return __builtin_bit_cast(float, (lane & 16) ? r[0] : r[1]);
}

// One layer's pages as the kernels see them.
struct cache_view {
	uint16_t* k;
	uint16_t* v;
	int64_t page_values; // values of one page: kv_heads * page_size * head_dim
	int pages;
	int kv_heads;
	int page_shift; // log2(page_size)
};
struct batch_view {
	const int32_t* table;
	const int32_t* lengths;
	const int32_t* starts;
	int sequences;
	int width;
};

// The sequence that packed row `row` belongs to: the b with starts[b] <= row < starts[b + 1], -1 if there is none.  starts ascends; an empty
// sequence shares its start with the next one and is passed over.
__device__ __forceinline__ int sequence_of_row(const int32_t* starts, int sequences, int row) {
	int lo = 0, hi = sequences + 1; // the first index whose start is above row lies in [lo, hi]
	while (lo < hi) {
		const int mid = (lo + hi) >> 1;
		if (starts[mid] > row) {
			hi = mid;
		} else {
			lo = mid + 1;
		}
	}
	return lo > 0 && lo <= sequences ? lo - 1 : -1;
}

// Softmax weights are formed as 2^(t - m + bias), t = scale log2(e) q.k, m what the row's weights are kept below: sums and products carry the same factor, which
// the last division takes out.  In the rows kernel m is the running maximum of t: fp16 weights lie in (0, 2^8] and keep all their bits down to 2^-22 of the
// largest.  In the tile kernel the maximum may have risen above m by up to `weight_rise` powers of two without being followed: fp16 weights lie in (0, 2^15].  (m is
// an fp32 number: t - m is off by up to 2^-24 |m|, so what is said here holds for scores of up to 2^23.)
template<int CACHE> constexpr float weight_bias = CACHE == NH_F16 ? 8.0f : 0.0f;
constexpr float weight_rise = 7.0f;
static_assert(weight_bias<NH_F16> + weight_rise < 16.0f, "a weight above 65504 is infinite in fp16");
constexpr float LOG2_E = 1.44269504088896340736f;

// Eight consecutive values of a q row as fp32 (all zero where there is no row).
template<int TYPE> __device__ __forceinline__ void load_q8(const void* q, int64_t at, bool there, float (&x)[8]) {
	if (!there) {
#pragma unroll
		for (int j = 0; j < 8; ++j) {
			x[j] = 0.0f;
		}
		return;
	}
	if constexpr (TYPE == NH_F32) {
		const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(q) + at);
		const float4 a = p[0], b = p[1];
		x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
	} else {
		const auto v = *reinterpret_cast<const typename half_type<TYPE>::vec*>(static_cast<const uint16_t*>(q) + at);
#pragma unroll
		for (int j = 0; j < 8; ++j) {
			x[j] = static_cast<float>(v[j]);
		}
	}
}
// The power of two that brings a row of fp32 q values, the largest of them `largest`, into the middle of fp16's range: q * 2^(14 - e) with
// 2^(e-1) <= largest < 2^e, so that two fp16 terms hold 22 bits of each value that matters beside the largest.  bf16 has fp32's range: e = 14.
template<int CACHE, int TYPE> __device__ __forceinline__ int q_exponent(float largest) {
	if constexpr (CACHE == NH_F16 && TYPE == NH_F32) {
		return max(__builtin_amdgcn_frexp_expf(largest), -60); // (0 for zero, infinity and NaN; a row smaller than 2^-60 gives scores of 2^-60: what is lost of it does not show)
	}
	return 14;
}

// Four values of an output row, rounded once.
template<int TYPE> __device__ __forceinline__ void store_out4(void* out, int64_t at, float a, float b, float c, float d) {
	if constexpr (TYPE == NH_F32) {
		*reinterpret_cast<float4*>(static_cast<float*>(out) + at) = make_float4(a, b, c, d);
	} else {
		typedef typename half_type<TYPE>::value v4t __attribute__((ext_vector_type(4)));
		using value = typename half_type<TYPE>::value;
		const v4t v{ static_cast<value>(a), static_cast<value>(b), static_cast<value>(c), static_cast<value>(d) };
		*reinterpret_cast<v4t*>(static_cast<uint16_t*>(out) + at) = v;
	}
}

// Values that are infinite or NaN: in a product they reach rows that do not see their keys too, and make NaN of what ought to be infinite (a weight of zero,
// or the negative rest of a weight in several terms, times infinity).  A result that is not finite is therefore formed once more: this time such values
// are taken out of the tiles and noted here, for each column of V the first such key, and a row that sees that key adds the value at the end.
template<int D> struct not_finite {
	int first_key[3][D]; // of NaN, +inf, -inf
	__device__ __forceinline__ void clear(int thread, int threads) {
		for (int i = thread; i < 3 * D; i += threads) {
			(&first_key[0][0])[i] = INT_MAX;
		}
	}
	// takes them out of the first n of eight values of column d, keys key .. key + 7
	template<int CACHE> __device__ __forceinline__ void take(uint16_t* eight, int d, int key, int n) {
		constexpr unsigned E = CACHE == NH_F16 ? 0x7C00u : 0x7F80u;
#pragma unroll 1
		for (int x = 0; x < min(n, 8); ++x) {
			const unsigned h = eight[x];
			if ((h & E) == E) {
				atomicMin(&first_key[(h & (E ^ 0x7FFFu)) ? 0 : 1 + (h >> 15)][d], key + x);
				eight[x] = 0;
			}
		}
	}
	// what a row that sees the keys below `seen` adds to column d
	__device__ __forceinline__ float of(int d, int seen) const {
		const bool nan = first_key[0][d] < seen, plus = first_key[1][d] < seen, minus = first_key[2][d] < seen;
		return nan || (plus && minus) ? __builtin_nanf("") : plus ? __builtin_inff() : minus ? -__builtin_inff() : 0.0f;
	}
};

// ---- launch functions (after argument checks) ----

// a launch has fewer threads along its grid than this
constexpr int64_t GRID_THREADS = int64_t{ 1 } << 32;

struct append_args {
	cache_view cache;
	batch_view batch;
	const void *q, *k, *v;
	void* q_out;
	const double* turns;
	int64_t q_stride, k_stride, v_stride;
	int rows, q_heads, head_dim, pairs;
	bool interleaved;
};
bool append_rope_fits(int64_t rows, int64_t kv_heads); // one launch
hipError_t launch_append_rope(const append_args& a, int cache_type, int type, hipStream_t s);

struct attention_args {
	cache_view cache;
	batch_view batch;
	const void* q;
	void* out;
	int64_t q_stride;
	int rows, q_heads, head_dim;
	float scale;
	const int32_t* prefix_pages; // decode only
	int prefix_count;
	bool prefix_apart; // for all sequences at once, by the tile kernel; else each reads it with its own keys
	void* workspace;
	int32_t* counters;
};
// What a kernel takes of the caller's memory, in bytes: its workspace, and counters that are zero before and after every call.
struct attention_needs {
	int64_t workspace, counters;
};
// The tile kernel (attention_prompt.hip): 128 rows of a sequence at a time.
attention_needs attention_tiles_needs(int64_t rows, int64_t sequences, int64_t q_heads, int64_t kv_heads, int64_t head_dim);
bool attention_tiles_fit(int64_t rows, int64_t sequences, int64_t q_heads, int64_t kv_heads); // one launch
hipError_t launch_attention_tiles(const attention_args& a, int cache_type, int type, hipStream_t s);
// The part of a decode step over a prefix that all sequences share: the batch's rows as tiles, the keys in pieces.
struct prefix_cut {
	int64_t pieces, keys, row_tiles; // keys of a piece
};
prefix_cut plan_prefix(int64_t sequences, int64_t group, int64_t kv_heads, int64_t prefix_keys);
bool prefix_fits(const prefix_cut& cut, int64_t kv_heads); // one launch
// partial results [piece][sequence][q_head]: o unnormalised, ml the running maximum (log2) and the sum of the weights
hipError_t launch_attention_prefix(const attention_args& a, int cache_type, int type, const prefix_cut& cut, float* o, float2* ml, hipStream_t s);
// The rows kernel (attention_rows.hip): 16 rows of a sequence at a time, each wave's keys and values through LDS of its own, long sequences in pieces.
attention_needs attention_rows_needs(int64_t sequences, bool one_each, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t prefix_keys);
// whether all work, in steps of 32 keys, surely has a 32-bit number (table_keys: what a sequence's table has room for)
bool attention_rows_fit(int64_t rows, int64_t sequences, bool one_each, int64_t group, int64_t table_keys);
hipError_t launch_attention_rows(const attention_args& a, int cache_type, int type, hipStream_t s);
// Which of the two a prompt's rows take (attention_abi.hip).
bool prompt_by_rows(int64_t rows, int64_t sequences, int64_t q_heads, int64_t kv_heads);

struct pages_args {
	uint16_t *k, *v;
	int64_t page_bytes; // of the keys, or of the values, of one page in one layer
	int64_t layers;
	int pages;
	int page_shift;
	batch_view batch;
	const int32_t *parents, *grow; // step only
	int children;
	int32_t *new_table, *new_lengths, *info;
	void* workspace;
};
int64_t cache_pages_workspace(int64_t pages, int64_t sequences, int64_t width);
hipError_t launch_cache_step(const pages_args& a, hipStream_t s);
hipError_t launch_cache_compact(const pages_args& a, hipStream_t s);

} // namespace nh
