// y [M][N] = x . w^T (+ residual) for int8 matrices with a scale per row, gfx950:  y[m][n] = sx[m] sw[n] sum_k x[m][k] w[n][k]
//
// The sums are whole numbers and exact (K is limited so that they stay below 2^31); each is brought to fp32, scaled by the row's and then by the channel's scale, the residual added,
// and rounded once to y's type.  The kernels are in i8_product.h.
#include "i8_product.h"

namespace nh {

namespace {

template<int TYPE> struct i8_store {
	typedef i8_type<TYPE> T;
	typedef typename T::store value;
	value* y;
	const value* residual;
	int M, N;

	template<int FN, int FM> __device__ __forceinline__ void operator()(const v4i (&sums)[FN][FM], int n0, int m0, const i8_matrix& w, const i8_matrix& x) const {
		const int lane = threadIdx.x & 63;
		const bool four = (N & 3) == 0; // then four neighbours lie together
#pragma unroll
		for (int i = 0; i < FM; ++i) {
			const int m = m0 + 16 * i + (lane & 15);
			if (m >= M) {
				continue;
			}
			const float sx = x.scale[m];
#pragma unroll
			for (int f = 0; f < FN; ++f) {
				const int n = n0 + 16 * f + 4 * (lane >> 4);
				if (n >= N) {
					continue;
				}
				const v4f sw	 = i8_scales4(w, n);
				const int64_t at = static_cast<int64_t>(m) * N + n;
				value out[4];
				float v[4];
#pragma unroll
				for (int e = 0; e < 4; ++e) {
					v[e] = static_cast<float>(sums[f][i][e]) * sx * sw[e];
				}
				if (four) {
					if (residual) {
						__builtin_memcpy(out, __builtin_assume_aligned(residual + at, 4 * sizeof(value)), sizeof(out));
#pragma unroll
						for (int e = 0; e < 4; ++e) {
							v[e] += T::widen(out[e]);
						}
					}
#pragma unroll
					for (int e = 0; e < 4; ++e) {
						out[e] = T::narrow(v[e]);
					}
					__builtin_memcpy(__builtin_assume_aligned(y + at, 4 * sizeof(value)), out, sizeof(out));
					continue;
				}
#pragma unroll
				for (int e = 0; e < 4; ++e) {
					if (n + e < N) {
						y[at + e] = T::narrow(residual ? v[e] + T::widen(residual[at + e]) : v[e]);
					}
				}
			}
		}
	}
};

template<int FN, int FM, int UNROLL, int TYPE> void rows_product(const i8_matrix& w, const i8_matrix& x, const i8_store<TYPE>& epi, hipStream_t stream) {
	const int n_tiles = (w.strips + FN - 1) / FN, m_tiles = (x.strips + FM - 1) / FM;
	i8_rows_product<FN, FM, UNROLL, 1><<<i8_grid(n_tiles, m_tiles), 512, 0, stream>>>(w, x, 0, n_tiles, m_tiles, epi);
}
template<int TYPE> hipError_t gemm(const i8_matrix& w, const i8_matrix& x, const void* residual, void* y, hipStream_t stream) {
	typedef typename i8_type<TYPE>::store value;
	const i8_store<TYPE> epi{ static_cast<value*>(y), static_cast<const value*>(residual), x.rows, w.rows };
	if (x.rows <= 16) {
		rows_product<1, 1, 8>(w, x, epi, stream);
	} else if (x.rows <= 32) {
		rows_product<2, 2, 4>(w, x, epi, stream);
	} else if (static_cast<int64_t>((x.rows + 255) / 256) * ((w.rows + 255) / 256) < 128) {
		rows_product<4, 4, 2>(w, x, epi, stream);
	} else {
		const int n_tiles = (w.rows + 255) / 256, m_tiles = (x.rows + 255) / 256;
		i8_tile_product<2, 4, 8, 4><<<i8_grid(n_tiles, m_tiles), 512, 0, stream>>>(w, x, 0, n_tiles, m_tiles, epi);
	}
	return hipGetLastError();
}

} // namespace

hipError_t launch_i8_gemm(const i8_matrix& w, const i8_matrix& x, const void* residual, void* y, int type, hipStream_t stream) {
	return type == NH_F32 ? gemm<NH_F32>(w, x, residual, y, stream) : type == NH_F16 ? gemm<NH_F16>(w, x, residual, y, stream) : gemm<NH_BF16>(w, x, residual, y, stream);
}

} // namespace nh
