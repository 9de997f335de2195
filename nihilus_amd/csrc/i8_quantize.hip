// Rows of activations (as they are, behind an RMS norm, or silu(gate) * up) to int8 with one scale per row, and plain int8 matrices into the tiled layout and back, gfx950.
//
//   s = fl32(max_j |v_j| / 127),  q_j = the whole number nearest to v_j / s, ties to even, within +-127
//
// s is a 32-bit float, and the quotient is the true one of the 32-bit floats v_j and s: whoever works it out in any way gets these numbers.  A row of zeros has s = 0 and
// q = 0; a row with an infinity or NaN has s = NaN and q = 0, so that whatever is formed from it is NaN, and nothing else is.
// v of a norm: fl32(fl32(x r) w), r = fl32(1 / sqrt(mean x^2 + eps)) with the mean in 64 bits, where the order of the sum does not show.
//
// Bound by memory.  A workgroup has four rows, 64 or 256 threads to a row, a thread sixteen values at a time (one 16-byte piece of a fragment), up to 64 of them kept in registers
// between the passes that a row's maximum and a norm need; longer rows are read again, from the caches.  The four workgroups of a strip go to one XCD, whose L2 joins their
// pieces to whole lines.
#include "i8_device.h"

namespace nh {

namespace {

constexpr int ROWS = 4; // of a workgroup
constexpr int HELD = 4; // pieces of sixteen values that a thread keeps

template<int TYPE> __device__ __forceinline__ void load16(const void* base, int64_t at, int left, bool wide, float (&v)[16]) {
	using T					  = i8_type<TYPE>;
	const auto* p			  = static_cast<const typename T::store*>(base) + at;
	constexpr int PER		  = 16 / sizeof(typename T::store);
	if (wide && left >= 16) {
#pragma unroll
		for (int i = 0; i < 16 / PER; ++i) {
			typename T::store part[PER];
			const v4u raw = *reinterpret_cast<const v4u*>(p + PER * i);
			__builtin_memcpy(part, &raw, 16);
#pragma unroll
			for (int j = 0; j < PER; ++j) {
				v[PER * i + j] = T::widen(part[j]);
			}
		}
		return;
	}
#pragma unroll
	for (int j = 0; j < 16; ++j) {
		v[j] = j < left ? T::widen(p[j]) : 0.0f;
	}
}

// The nearest whole number to v / s.  c is one of the two next to the quotient; v - c s is exact wherever it is close to half of s (a difference of multiples of the last place
// of the smaller of v and s, below s), so comparing it with s / 2 decides between the two.
__device__ __forceinline__ int nearest(float v, float s, float inverse) {
	float c		  = rintf(v * inverse);
	const float e = fmaf(-c, s, v), half = 0.5f * s;
	if (fabsf(e) >= half && (fabsf(e) > half || (static_cast<int>(c) & 1))) {
		c += copysignf(1.0f, e);
	}
	return static_cast<int>(fminf(fmaxf(c, -127.0f), 127.0f));
}

template<int TYPE, int FRONT, int THREADS> __global__ __launch_bounds__(ROWS* THREADS) void i8_quantize_kernel(i8_rows in, v4u* q, float* scale, int steps, bool wide, bool wide_up) {
	constexpr int WAVES = THREADS / 64; // of a row
	__shared__ double sums[ROWS][WAVES];
	__shared__ uint32_t tops[ROWS][WAVES];
	const int i	  = blockIdx.x >> 3;
	const int row = ((i >> 2) * 8 + (blockIdx.x & 7)) * I8_ROWS + ROWS * (i & 3) + threadIdx.x / THREADS;
	const int mine = threadIdx.x / THREADS, t = threadIdx.x % THREADS, wave = t >> 6;
	const bool there = row < in.rows;
	const int pieces = there ? 4 * steps : 0;
	const int64_t at = static_cast<int64_t>(row) * in.stride, up_at = static_cast<int64_t>(row) * in.up_stride;
	float r = 1.0f;
	auto get = [&](int c, float(&v)[16]) { // without the norm
		load16<TYPE>(in.x, at + 16 * c, in.k - 16 * c, wide, v);
		if constexpr (FRONT == I8_SILU) {
			float u[16];
			load16<TYPE>(in.up, up_at + 16 * c, in.k - 16 * c, wide_up, u);
#pragma unroll
			for (int j = 0; j < 16; ++j) {
				v[j] = silu_mul(v[j], u[j]);
			}
		}
	};
	auto normed = [&](int c, float(&v)[16]) {
		if constexpr (FRONT == I8_NORM) {
			float w[16];
			load16<NH_F32>(in.norm, 16 * c, in.k - 16 * c, true, w);
#pragma unroll
			for (int j = 0; j < 16; ++j) {
				v[j] = __fmul_rn(__fmul_rn(v[j], r), w[j]);
			}
		}
	};
	float held[HELD][16];
#pragma unroll
	for (int h = 0; h < HELD; ++h) {
		if (t + THREADS * h < pieces) {
			get(t + THREADS * h, held[h]);
		}
	}
	if constexpr (FRONT == I8_NORM) {
		double sum = 0.0;
		auto add   = [&](const float(&v)[16]) {
#pragma unroll
			for (int j = 0; j < 16; ++j) {
				sum = fma(static_cast<double>(v[j]), static_cast<double>(v[j]), sum);
			}
		};
#pragma unroll
		for (int h = 0; h < HELD; ++h) {
			if (t + THREADS * h < pieces) {
				add(held[h]);
			}
		}
		for (int c = t + THREADS * HELD; c < pieces; c += THREADS) {
			float v[16];
			get(c, v);
			add(v);
		}
#pragma unroll
		for (int d = 32; d > 0; d >>= 1) {
			sum += __shfl_xor(sum, d);
		}
		if constexpr (WAVES > 1) {
			if ((t & 63) == 0) {
				sums[mine][wave] = sum;
			}
			__syncthreads();
			sum = sums[mine][0];
#pragma unroll
			for (int w = 1; w < WAVES; ++w) {
				sum += sums[mine][w];
			}
		}
		r = static_cast<float>(1.0 / sqrt(sum / in.k + static_cast<double>(in.eps)));
	}
	uint32_t top = 0; // of the values' bits without their signs: infinities and NaN are above all others
	auto raise	 = [&](const float(&v)[16]) {
#pragma unroll
		for (int j = 0; j < 16; ++j) {
			top = max(top, __float_as_uint(v[j]) & 0x7FFFFFFFu);
		}
	};
#pragma unroll
	for (int h = 0; h < HELD; ++h) {
		if (t + THREADS * h < pieces) {
			normed(t + THREADS * h, held[h]);
			raise(held[h]);
		}
	}
	for (int c = t + THREADS * HELD; c < pieces; c += THREADS) {
		float v[16];
		get(c, v);
		normed(c, v);
		raise(v);
	}
#pragma unroll
	for (int d = 32; d > 0; d >>= 1) {
		top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), d)));
	}
	if constexpr (WAVES > 1) {
		if ((t & 63) == 0) {
			tops[mine][wave] = top;
		}
		__syncthreads();
#pragma unroll
		for (int w = 0; w < WAVES; ++w) {
			top = max(top, tops[mine][w]);
		}
	}
	const bool finite = top < 0x7F800000u;
	const float s	  = finite ? __fdiv_rn(__uint_as_float(top), 127.0f) : __builtin_nanf("");
	if (there && t == 0) {
		scale[row] = s;
	}
	// far down both are brought up, which is exact, so that the reciprocal and the products stay normal numbers
	const float lift	= s < 0x1p-100f ? 0x1p100f : 1.0f;
	const float step	= s * lift;
	const bool nothing	= !finite || s == 0.0f;
	const float inverse = nothing ? 0.0f : __builtin_amdgcn_rcpf(step);
	auto put			= [&](int c, const float(&v)[16]) {
		   v4u out;
#pragma unroll
		   for (int d = 0; d < 4; ++d) {
			   uint32_t word = 0;
#pragma unroll
			   for (int j = 0; j < 4; ++j) {
				   word |= (static_cast<uint32_t>(nearest(v[4 * d + j] * lift, step, inverse)) & 0xFFu) << (8 * j);
			   }
			   out[d] = nothing ? 0u : word;
		   }
		   q[(static_cast<int64_t>(row >> 4) * steps + (c >> 2)) * 64 + (c & 3) * 16 + (row & 15)] = out;
	};
#pragma unroll
	for (int h = 0; h < HELD; ++h) {
		if (t + THREADS * h < pieces) {
			put(t + THREADS * h, held[h]);
		}
	}
	for (int c = t + THREADS * HELD; c < pieces; c += THREADS) {
		float v[16];
		get(c, v);
		normed(c, v);
		put(c, v);
	}
}

// one 16-byte piece of a fragment per thread
__global__ __launch_bounds__(256) void i8_tile_kernel(const int8_t* q, const float* scales, v4u* out, float* out_scales, int64_t rows, int64_t k, int64_t strips, int64_t steps) {
	const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
	if (i < strips * I8_ROWS) {
		out_scales[i] = i < rows ? scales[i] : 0.0f;
	}
	if (i >= strips * steps * 64) {
		return;
	}
	const int lane	  = i & 63;
	const int64_t row = (i >> 6) / steps * I8_ROWS + (lane & 15), at = (i >> 6) % steps * I8_STEP + 16 * (lane >> 4);
	uint32_t word[4]  = {};
	if (row < rows) {
#pragma unroll
		for (int j = 0; j < 16; ++j) {
			if (at + j < k) {
				word[j / 4] |= static_cast<uint32_t>(static_cast<uint8_t>(q[row * k + at + j])) << (8 * (j % 4));
			}
		}
	}
	out[i] = v4u{ word[0], word[1], word[2], word[3] };
}

__global__ __launch_bounds__(256) void i8_untile_kernel(const v4u* in, const float* in_scales, int8_t* q, float* scales, int64_t rows, int64_t k, int64_t strips, int64_t steps) {
	const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
	if (i < rows) {
		scales[i] = in_scales[i];
	}
	if (i >= strips * steps * 64) {
		return;
	}
	const int lane	  = i & 63;
	const int64_t row = (i >> 6) / steps * I8_ROWS + (lane & 15), at = (i >> 6) % steps * I8_STEP + 16 * (lane >> 4);
	if (row < rows) {
		const v4u v = in[i];
#pragma unroll
		for (int j = 0; j < 16; ++j) {
			if (at + j < k) {
				q[row * k + at + j] = static_cast<int8_t>(v[j / 4] >> (8 * (j % 4)));
			}
		}
	}
}

template<int TYPE, int FRONT> hipError_t quantize(const i8_rows& in, v4u* q, float* scale, int steps, hipStream_t stream) {
	constexpr int64_t size = sizeof(typename i8_type<TYPE>::store);
	auto apart			   = [&](const void* p, int64_t stride) {
		return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && stride * size % 16 == 0;
	};
	const bool wide	 = apart(in.x, in.stride), wide_up = FRONT == I8_SILU && apart(in.up, in.up_stride);
	const int blocks = static_cast<int>((i8_strips(in.rows) + 7) / 8) * 32;
	i8_quantize_kernel<TYPE, FRONT, 256><<<blocks, ROWS * 256, 0, stream>>>(in, q, scale, steps, wide, wide_up);
	return hipGetLastError();
}
template<int TYPE> hipError_t quantize(const i8_rows& in, int front, v4u* q, float* scale, int steps, hipStream_t stream) {
	return front == I8_NORM ? quantize<TYPE, I8_NORM>(in, q, scale, steps, stream)
		: front == I8_SILU	? quantize<TYPE, I8_SILU>(in, q, scale, steps, stream)
							: quantize<TYPE, I8_PLAIN>(in, q, scale, steps, stream);
}

} // namespace

hipError_t launch_i8_quantize(const i8_rows& in, int front, int type, void* tiled, hipStream_t stream) {
	const i8_matrix m = i8_view(tiled, in.rows, in.k);
	v4u* q			  = static_cast<v4u*>(tiled);
	float* scale	  = const_cast<float*>(m.scale);
	return type == NH_F32 ? quantize<NH_F32>(in, front, q, scale, m.steps, stream)
		: type == NH_F16  ? quantize<NH_F16>(in, front, q, scale, m.steps, stream)
						  : quantize<NH_BF16>(in, front, q, scale, m.steps, stream);
}

hipError_t launch_i8_tile(const int8_t* q, const float* scales, void* tiled, int64_t rows, int64_t k, hipStream_t stream) {
	const i8_matrix m	 = i8_view(tiled, rows, k);
	const int64_t pieces = static_cast<int64_t>(m.strips) * m.steps * 64;
	i8_tile_kernel<<<static_cast<unsigned>((pieces + 255) / 256), 256, 0, stream>>>(q, scales, static_cast<v4u*>(tiled), const_cast<float*>(m.scale), rows, k, m.strips, m.steps);
	return hipGetLastError();
}

hipError_t launch_i8_untile(const void* tiled, int8_t* q, float* scales, int64_t rows, int64_t k, hipStream_t stream) {
	const i8_matrix m	 = i8_view(tiled, rows, k);
	const int64_t pieces = static_cast<int64_t>(m.strips) * m.steps * 64;
	i8_untile_kernel<<<static_cast<unsigned>((pieces + 255) / 256), 256, 0, stream>>>(m.q, m.scale, q, scales, rows, k, m.strips, m.steps);
	return hipGetLastError();
}

} // namespace nh
