// Values of activations and the whole numbers nearest to them in units of a row's scale.
#pragma once

#include "i8_device.h"

namespace nh {

// N values (8 or 16); those from `left` on are zero (rows begin anywhere: the hardware takes any address)
template<int TYPE, int N> __device__ __forceinline__ void i8_load(const void* base, int64_t at, int left, float (&v)[N]) {
	using T		  = i8_type<TYPE>;
	const auto* p = static_cast<const typename T::store*>(base) + at;
	if (left >= N) {
		typename T::store part[N];
		__builtin_memcpy(part, p, sizeof(part));
#pragma unroll
		for (int j = 0; j < N; ++j) {
			v[j] = T::widen(part[j]);
		}
		return;
	}
#pragma unroll
	for (int j = 0; j < N; ++j) {
		v[j] = j < left ? T::widen(p[j]) : 0.0f;
	}
}

// The whole numbers nearest to v / s as bytes, `inverse` being 1 / s to a unit in the last place.  c, the product with that rounded, is one of the two next to the quotient, and v - c s is
// exact wherever it is close to half of s (a difference of multiples of the last place of the smaller of v and s, below s): comparing it with s / 2 decides between the two.  Where no
// value of the wave's is that close, which is nearly always, c is right as it is.
// (`doubt`: they may be past 127, which rows below the normal numbers reach, whose scale has few bits)
template<int N> __device__ __forceinline__ void i8_nearest(const float (&v)[N], float s, float inverse, bool doubt, uint32_t (&out)[N / 4]) {
	constexpr float magic = 12582912.0f; // 1.5 * 2^23: the sum's low byte is the whole number
	float c[N], far = 0.0f;
#pragma unroll
	for (int j = 0; j < N; ++j) {
		c[j] = fmaf(v[j], inverse, magic);
		far	 = fmaxf(far, fabsf(fmaf(magic - c[j], s, v[j])));
	}
	if (doubt || far >= 0.5f * s) {
#pragma unroll
		for (int j = 0; j < N; ++j) {
			float n		  = c[j] - magic;
			const float e = fmaf(-n, s, v[j]), half = 0.5f * s;
			if (fabsf(e) >= half && (fabsf(e) > half || (static_cast<int>(n) & 1))) {
				n += copysignf(1.0f, e);
			}
			c[j] = fminf(fmaxf(n, -127.0f), 127.0f) + magic;
		}
	}
#pragma unroll
	for (int d = 0; d < N / 4; ++d) { // (selector: 0..3 bytes of the second operand, 4..7 of the first)
		const uint32_t low	= __builtin_amdgcn_perm(__float_as_uint(c[4 * d + 1]), __float_as_uint(c[4 * d]), 0x0c0c0400u);
		const uint32_t high = __builtin_amdgcn_perm(__float_as_uint(c[4 * d + 3]), __float_as_uint(c[4 * d + 2]), 0x04000c0cu);
		out[d]				= low | high;
	}
}

// A row's scale from the bits of its largest value without signs (infinities and NaN are above all others), and what i8_nearest wants of it: s = fl32(top / 127), NaN if the row is not finite;
// far down both the values and s are brought up by 2^100, which is exact, so that the reciprocal and the products stay normal numbers.
struct i8_step {
	float scale, step, inverse, lift;
	bool nothing; // zeros whatever the values are

	__device__ __forceinline__ explicit i8_step(uint32_t top) {
		const bool finite = top < 0x7F800000u;
		scale			  = finite ? __fdiv_rn(__uint_as_float(top), 127.0f) : __builtin_nanf("");
		lift			  = scale < 0x1p-100f ? 0x1p100f : 1.0f;
		step			  = scale * lift;
		nothing			  = !finite || scale == 0.0f;
		inverse			  = nothing ? 0.0f : __builtin_amdgcn_rcpf(step);
	}
	template<int N> __device__ __forceinline__ void round(float (&v)[N], uint32_t (&out)[N / 4]) const {
		if (lift != 1.0f) {
#pragma unroll
			for (int j = 0; j < N; ++j) {
				v[j] *= lift;
			}
		}
		i8_nearest(v, step, inverse, lift != 1.0f, out);
		if (nothing) {
#pragma unroll
			for (int d = 0; d < N / 4; ++d) {
				out[d] = 0;
			}
		}
	}
};
// 1 / rms of a row as the norm wants it, from the sum of its squares and 1 / k
__device__ __forceinline__ float i8_rms(double sum, double part, float eps) {
	return static_cast<float>(rsqrt(fma(sum, part, static_cast<double>(eps))));
}

} // namespace nh
