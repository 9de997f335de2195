// Rope on q and k and the write of k and v into the paged cache, one launch, gfx950.
//
//   theta = 2 pi turns[i] p,  (a, b) -> (a cos theta - b sin theta, a sin theta + b cos theta)
//
// (rope and cache write of the reference's mega_qkv core, infra/core_traits.hpp:596-616, whose GPU body is empty.)
//
// Angles: turns[i] * p is formed in fp64 and only its fractional part goes on in fp32: at position 10^5 an fp32 product has lost all but
// seven bits of the fraction, the fp64 one keeps 36.  sin and cos of the part, and the rotation, are fp32 (1e-7 relative); the result is rounded once.
//
// Memory-bound.  A thread owns the same two pairs of every head that it touches, so their sines are worked out once per thread and row,
// without a table and without a barrier.  Many rows: one workgroup per row; few rows: the heads of a row over several workgroups, for latency.
// v is transposed inside its page, 64 rows at a time through LDS, so that consecutive lanes write consecutive tokens.
// Measured: prompts of up to 3001 rows of 64 query heads over 8 kv heads of 128, fp32 to fp16, 552 MB, take 112 us, 4.9 TB/s, the rate of a large copy; one row 4.9 us with its call, the kernel 3.1 to 3.3, an empty launch 2.3.
#include "attention_device.h"

namespace nh {

namespace {

constexpr int THREADS = 256;
constexpr int V_ROWS  = 64;

template<int TYPE> struct io;
template<> struct io<NH_F32> {
	static __device__ __forceinline__ float2 load2(const void* p, int64_t i) {
		return *reinterpret_cast<const float2*>(static_cast<const float*>(p) + i);
	}
	static __device__ __forceinline__ void store2(void* p, int64_t i, float2 v) {
		*reinterpret_cast<float2*>(static_cast<float*>(p) + i) = v;
	}
};
template<> struct io<NH_F16> {
	static __device__ __forceinline__ float2 load2(const void* p, int64_t i) {
		return __half22float2(*reinterpret_cast<const __half2*>(static_cast<const __half*>(p) + i));
	}
	static __device__ __forceinline__ void store2(void* p, int64_t i, float2 v) {
		*reinterpret_cast<__half2*>(static_cast<__half*>(p) + i) = __float22half2_rn(v);
	}
};
template<> struct io<NH_BF16> {
	static __device__ __forceinline__ float2 load2(const void* p, int64_t i) {
		const uint32_t u = *reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(p) + i);
		return make_float2(__builtin_bit_cast(float, u << 16), __builtin_bit_cast(float, u & 0xFFFF0000u));
	}
	static __device__ __forceinline__ void store2(void* p, int64_t i, float2 v) {
		typedef __bf16 v2b __attribute__((ext_vector_type(2)));
		const v2b b{ static_cast<__bf16>(v.x), static_cast<__bf16>(v.y) };
		*reinterpret_cast<v2b*>(static_cast<uint16_t*>(p) + i) = b;
	}
};

// position of a packed row in its sequence and that sequence; false for a row that no sequence has
__device__ __forceinline__ bool place_of_row(const batch_view& b, int row, int& seq, int& pos) {
	if (b.starts) {
		seq = sequence_of_row(b.starts, b.sequences, row);
		if (seq < 0) {
			return false;
		}
		pos = max(b.lengths[seq], 0) - (b.starts[seq + 1] - row);
		return true;
	}
	seq = row;
	pos = max(b.lengths[row], 0) - 1;
	return true;
}
// the page of a position, or -1
__device__ __forceinline__ int page_of(const batch_view& b, const cache_view& c, int seq, int pos) {
	const int slot = pos >> c.page_shift;
	if (pos < 0 || slot >= b.width) {
		return -1;
	}
	const int id = b.table[static_cast<int64_t>(seq) * b.width + slot];
	return id >= 0 && id < c.pages ? id : -1;
}

} // namespace

template<int CACHE, int TYPE, int D, bool INTERLEAVED>
__global__ __launch_bounds__(THREADS) void append_rope_kernel(append_args a, int chunks, int rotate_blocks) {
	constexpr int PER_HEAD = D / 4; // threads of a head: two pairs each
	constexpr int HEADS	   = THREADS / PER_HEAD; // heads side by side
	const int page_size	   = 1 << a.cache.page_shift;
	if (static_cast<int>(blockIdx.x) < rotate_blocks) {
		const int row = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
		int seq, pos;
		if (!place_of_row(a.batch, row, seq, pos)) {
			return;
		}
		const int c	 = threadIdx.x % PER_HEAD;
		const bool turned = 2 * c < a.pairs;
		// where this thread's four values lie in a head
		const int e0 = INTERLEAVED ? 4 * c : turned ? 2 * c : 2 * a.pairs + 4 * (c - a.pairs / 2);
		const int e1 = !INTERLEAVED && turned ? e0 + a.pairs : e0 + 2;
		float sin0 = 0.0f, cos0 = 1.0f, sin1 = 0.0f, cos1 = 1.0f;
		if (turned) {
			const double t0 = a.turns[2 * c] * static_cast<double>(pos), t1 = a.turns[2 * c + 1] * static_cast<double>(pos);
			sincospif(2.0f * static_cast<float>(t0 - rint(t0)), &sin0, &cos0);
			sincospif(2.0f * static_cast<float>(t1 - rint(t1)), &sin1, &cos1);
		}
		const int page		  = page_of(a.batch, a.cache, seq, pos);
		const int heads		  = a.q_heads + a.cache.kv_heads;
		const int64_t q_row	  = row * a.q_stride, k_row = row * a.k_stride, out_row = static_cast<int64_t>(row) * a.q_heads * D;
		for (int h = chunk * HEADS + threadIdx.x / PER_HEAD; h < heads; h += chunks * HEADS) {
			const bool is_q	   = h < a.q_heads;
			const void* src	   = is_q ? a.q : a.k;
			const int64_t from = is_q ? q_row + static_cast<int64_t>(h) * D : k_row + static_cast<int64_t>(h - a.q_heads) * D;
			float2 x = io<TYPE>::load2(src, from + e0), y = io<TYPE>::load2(src, from + e1);
			if (turned) {
				if constexpr (INTERLEAVED) { // pairs (x.x, x.y), (y.x, y.y)
					x = make_float2(x.x * cos0 - x.y * sin0, x.x * sin0 + x.y * cos0);
					y = make_float2(y.x * cos1 - y.y * sin1, y.x * sin1 + y.y * cos1);
				} else { // pairs (x.x, y.x), (x.y, y.y)
					const float2 u = make_float2(x.x * cos0 - y.x * sin0, x.y * cos1 - y.y * sin1);
					y			   = make_float2(x.x * sin0 + y.x * cos0, x.y * sin1 + y.y * cos1);
					x			   = u;
				}
			}
			if (is_q) {
				io<TYPE>::store2(a.q_out, out_row + static_cast<int64_t>(h) * D + e0, x);
				io<TYPE>::store2(a.q_out, out_row + static_cast<int64_t>(h) * D + e1, y);
			} else if (page >= 0) {
				const int64_t to = page * a.cache.page_values + (static_cast<int64_t>(h - a.q_heads) * page_size + (pos & (page_size - 1))) * D;
				io<CACHE>::store2(a.cache.k, to + e0, x);
				io<CACHE>::store2(a.cache.k, to + e1, y);
			}
		}
		return;
	}
	// v: rows r0 .. r0 + n - 1 of one head
	__shared__ uint32_t tile[V_ROWS][D / 2 + 1]; // (one more: lanes that read a column hit different banks)
	__shared__ int64_t where[V_ROWS]; // first value of the row's place in the V pages, or -1
	const int b	 = blockIdx.x - rotate_blocks;
	const int h	 = b % a.cache.kv_heads;
	const int r0 = (b / a.cache.kv_heads) * V_ROWS;
	const int n	 = min(V_ROWS, a.rows - r0);
	if (static_cast<int>(threadIdx.x) < n) {
		int seq, pos;
		int64_t at = -1;
		if (place_of_row(a.batch, r0 + threadIdx.x, seq, pos)) {
			const int page = page_of(a.batch, a.cache, seq, pos);
			if (page >= 0) {
				at = page * a.cache.page_values + static_cast<int64_t>(h) * D * page_size + (pos & (page_size - 1));
			}
		}
		where[threadIdx.x] = at;
	}
	__syncthreads();
	for (int i = threadIdx.x; i < n * (D / 2); i += THREADS) {
		const int r = i / (D / 2), c = i % (D / 2);
		if (where[r] >= 0) { // (rows of nobody are not read either)
			io<CACHE>::store2(&tile[r][c], 0, io<TYPE>::load2(a.v, (r0 + r) * a.v_stride + static_cast<int64_t>(h) * D + 2 * c));
		}
	}
	__syncthreads();
	for (int i = threadIdx.x; i < n * D; i += THREADS) {
		const int d = i / n, r = i % n;
		if (where[r] >= 0) {
			a.cache.v[where[r] + static_cast<int64_t>(d) * page_size] = reinterpret_cast<const uint16_t*>(&tile[r][0])[d];
		}
	}
}

// (with the heads of a row over several workgroups there are 2048 of those at most)
bool append_rope_fits(int64_t rows, int64_t kv_heads) {
	return (rows + (rows + V_ROWS - 1) / V_ROWS * kv_heads) * THREADS < GRID_THREADS;
}

template<int CACHE, int TYPE, int D> static hipError_t launch_append(const append_args& a, hipStream_t s) {
	constexpr int HEADS = THREADS / (D / 4);
	const int64_t full	= (a.q_heads + a.cache.kv_heads + HEADS - 1) / HEADS;
	// a row's heads side by side as long as that does not give more workgroups than the chip holds at once
	const int64_t chunks = a.rows * full <= 2048 ? full : 1;
	const int64_t rotate = a.rows * chunks, v = (a.rows + V_ROWS - 1) / V_ROWS * a.cache.kv_heads;
	const dim3 grid(static_cast<unsigned>(rotate + v));
	if (a.interleaved) {
		append_rope_kernel<CACHE, TYPE, D, true><<<grid, dim3(THREADS), 0, s>>>(a, static_cast<int>(chunks), static_cast<int>(rotate));
	} else {
		append_rope_kernel<CACHE, TYPE, D, false><<<grid, dim3(THREADS), 0, s>>>(a, static_cast<int>(chunks), static_cast<int>(rotate));
	}
	return hipGetLastError();
}
template<int CACHE, int TYPE> static hipError_t launch_append(const append_args& a, hipStream_t s) {
	return a.head_dim == 64 ? launch_append<CACHE, TYPE, 64>(a, s) : launch_append<CACHE, TYPE, 128>(a, s);
}

hipError_t launch_append_rope(const append_args& a, int cache_type, int type, hipStream_t s) {
	if (cache_type == NH_F16) {
		return type == NH_F32 ? launch_append<NH_F16, NH_F32>(a, s) : launch_append<NH_F16, NH_F16>(a, s);
	}
	return type == NH_F32 ? launch_append<NH_BF16, NH_F32>(a, s) : launch_append<NH_BF16, NH_BF16>(a, s);
}

} // namespace nh
