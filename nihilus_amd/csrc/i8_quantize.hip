// Rows of activations (as they are, behind an RMS norm, or silu(gate) * up) to int8 with one scale per row, and plain int8 matrices into the tiled layout and back, gfx950.
//
//   s = fl32(max_j |v_j| / 127),  q_j = the whole number nearest to v_j / s, ties to even, within +-127
//
// s is a 32-bit float, and the quotient is the true one of the 32-bit floats v_j and s: whoever works it out in any way gets these numbers.  A row of zeros has s = 0 and
// q = 0; a row with an infinity or NaN has s = NaN and q = 0, so that whatever is formed from it is NaN, and nothing else is.
// v of a norm: fl32(fl32(x r) w), r = fl32(1 / sqrt(mean x^2 + eps)) with the mean in 64 bits, where the order of the sum does not show.
//
// Bound by memory where rows are many, by the chain of a row's passes where they are few: a workgroup has a row, a thread HELD pieces of sixteen values (16 bytes of a fragment each), which it
// keeps in registers between the passes that a row's maximum and a norm need; rows longer than that are read again, from the caches.  The sixteen workgroups of a strip go to one XCD,
// whose L2 joins their pieces to whole lines.
#include "i8_values.h"

namespace nh {

namespace {

// silu(g) u within 3 units of 2^-23 of itself, or of 2^-149.  -g log2(e) in two parts (the second brought in behind the exponential), the exponential's one unit, a sum, a quotient by one correction step (so
// within half a unit and little more), a product.  NEAR: |g| is up to 80 or NaN, where exp(-g), the sum and the quotient are normal numbers.  Above that 1 + exp(-g) is 1; below -80 it is exp(-g), and the
// result g exp(g) u, formed 2^64 times as large: exp(g) is then a normal number down to g = -131, past which 0 is taken.
template<bool NEAR> __device__ __forceinline__ float silu_times(float g, float u) {
	constexpr float log2e = 1.44269502162933349609375f, log2e_rest = 1.925963033500011e-8f, ln2 = 0.693147182464599609375f;
	const bool far_down = !NEAR && g < -80.0f;
	const float held	= NEAR ? g : fminf(fmaxf(g, -256.0f), 80.0f), at = far_down ? held : -held;
	const float t		= at * log2e;
	const float rest	= fmaf(at, log2e, -t) + at * log2e_rest;
	float e				= __builtin_amdgcn_exp2f(far_down ? t + 64.0f : t); // (that sum is exact)
	e					= fmaf(e, rest * ln2, e);
	if (far_down) {
		return g * e * u * 0x1p-64f;
	}
	if (!NEAR && g > 80.0f) {
		return g * u;
	}
	const float d = 1.0f + e, r = __builtin_amdgcn_rcpf(d), q = g * r;
	return fmaf(fmaf(-q, d, g), r, q) * u;
}
template<int N> __device__ __forceinline__ void silu_times(float (&g)[N], const float (&u)[N]) {
	float far = 0.0f;
#pragma unroll
	for (int j = 0; j < N; ++j) {
		far = fmaxf(far, fabsf(g[j]));
	}
	if (far <= 80.0f) {
#pragma unroll
		for (int j = 0; j < N; ++j) {
			g[j] = silu_times<true>(g[j], u[j]);
		}
	} else {
#pragma unroll
		for (int j = 0; j < N; ++j) {
			g[j] = silu_times<false>(g[j], u[j]);
		}
	}
}

template<int TYPE, int FRONT, int THREADS, int HELD> __global__ __launch_bounds__(THREADS) void i8_quantize_kernel(i8_rows in, v4u* q, float* scale, int steps) {
	constexpr int WAVES = THREADS / 64; // of a row
	__shared__ double sums[WAVES];
	__shared__ uint32_t tops[WAVES];
	const int i	  = blockIdx.x >> 3;
	const int row = ((i >> 4) * 8 + (blockIdx.x & 7)) * I8_ROWS + (i & 15);
	const int t	  = threadIdx.x, wave = t >> 6;
	if (row >= in.rows) {
		return;
	}
	const int pieces = 4 * steps;
	const int64_t at = static_cast<int64_t>(row) * in.stride, up_at = static_cast<int64_t>(row) * in.up_stride;
	float r = 1.0f;
	auto get = [&](int c, float(&v)[16]) { // without the norm
		i8_load<TYPE>(in.x, at + 16 * c, in.k - 16 * c, v);
		if constexpr (FRONT == I8_SILU) {
			float u[16];
			i8_load<TYPE>(in.up, up_at + 16 * c, in.k - 16 * c, u);
			silu_times(v, u);
		}
	};
	auto normed = [&](int c, float(&v)[16]) {
		if constexpr (FRONT == I8_NORM) {
			float w[16];
			i8_load<NH_F32>(in.norm, 16 * c, in.k - 16 * c, w);
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
		if ((t & 63) == 0) {
			sums[wave] = sum;
		}
		__syncthreads();
		sum = sums[0];
#pragma unroll
		for (int w = 1; w < WAVES; ++w) {
			sum += sums[w];
		}
		r = i8_rms(sum, in.part, in.eps);
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
	if ((t & 63) == 0) {
		tops[wave] = top;
	}
	__syncthreads();
#pragma unroll
	for (int w = 0; w < WAVES; ++w) {
		top = max(top, tops[w]);
	}
	const i8_step step(top);
	if (t == 0) {
		scale[row] = step.scale;
	}
	auto put = [&](int c, float(&v)[16]) {
		uint32_t out[4];
		step.round(v, out);
		q[(static_cast<int64_t>(row >> 4) * steps + (c >> 2)) * 64 + (c & 3) * 16 + (row & 15)] = v4u{ out[0], out[1], out[2], out[3] };
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
	if (row < rows && at + 16 <= k) {
		__builtin_memcpy(word, q + row * k + at, 16);
	} else if (row < rows) {
		for (int j = 0; at + j < k; ++j) {
			word[j / 4] |= static_cast<uint32_t>(static_cast<uint8_t>(q[row * k + at + j])) << (8 * (j % 4));
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
		if (at + 16 <= k) {
			__builtin_memcpy(q + row * k + at, &v, 16);
		} else {
#pragma unroll
			for (int j = 0; j < 16; ++j) {
				if (at + j < k) {
					q[row * k + at + j] = static_cast<int8_t>(v[j / 4] >> (8 * (j % 4)));
				}
			}
		}
	}
}

template<int TYPE, int FRONT> hipError_t quantize(const i8_rows& in, v4u* q, float* scale, int steps, hipStream_t stream) {
	const unsigned blocks = static_cast<unsigned>((i8_strips(in.rows) + 7) / 8 * 8 * I8_ROWS);
	auto launch			  = [&](auto kernel, int threads) {
		kernel<<<blocks, threads, 0, stream>>>(in, q, scale, steps);
	};
	// Few rows: more threads to a row; many: fewer, so that more rows are under way.  us: 13 x 8192 bf16 3.8 by 512 threads, 5.0 by 256; 8192 x 8192 bf16 behind a norm 58 by 256, 71 by four rows of 256 threads to
	// a workgroup; silu of 512 x 14336 bf16 12.1 by 512 threads, 13.7 by 1024; of 8192 x 14336 128 by 256 threads, 169 by 1024.
	if (steps <= 64) {
		launch(i8_quantize_kernel<TYPE, FRONT, 256, 1>, 256);
	} else if (steps <= 128) {
		in.rows <= 1024 ? launch(i8_quantize_kernel<TYPE, FRONT, 512, 1>, 512) : launch(i8_quantize_kernel<TYPE, FRONT, 256, 2>, 256);
	} else if (steps <= 256) {
		in.rows <= 1024 ? launch(i8_quantize_kernel<TYPE, FRONT, 512, 2>, 512) : launch(i8_quantize_kernel<TYPE, FRONT, 256, 4>, 256);
	} else {
		launch(i8_quantize_kernel<TYPE, FRONT, 512, 4>, 512);
	}
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
