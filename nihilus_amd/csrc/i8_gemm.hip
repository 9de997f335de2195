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

	// A lane has four neighbouring n of sixteen different rows m: sixteen rows at a time go through LDS, so that a wave's stores run along the rows.  Pieces of four values lie at
	// places permuted by the row, which spreads them over the banks either way.
	template<int FN, int FM> __device__ __forceinline__ void operator()(const v4i (&sums)[FN][FM], int n0, int m0, const i8_matrix& w, const i8_matrix& x, v4f* scratch) const {
		constexpr int PIECES = 4 * FN; // of a row
		const int lane = threadIdx.x & 63, row = lane & 15;
		const bool fours = (N & 3) == 0; // then four neighbours lie together in y
#pragma unroll
		for (int i = 0; i < FM; ++i) {
			const int m	   = m0 + 16 * i;
			const float sx = m + row < M ? x.scale[m + row] : 0.0f;
#pragma unroll
			for (int f = 0; f < FN; ++f) {
				const int piece = 4 * f + (lane >> 4);
				const v4f sw	= i8_scales4(w, n0 + 4 * piece);
				v4f v;
#pragma unroll
				for (int e = 0; e < 4; ++e) {
					v[e] = static_cast<float>(sums[f][i][e]) * sx * sw[e];
				}
				scratch[row * PIECES + (piece ^ (row % PIECES))] = v;
			}
			__builtin_amdgcn_wave_barrier(); // (one wave's own LDS accesses are in order)
			if (fours) {
				constexpr int AT_ONCE = 64 / PIECES; // rows
#pragma unroll
				for (int r0 = 0; r0 < 16; r0 += AT_ONCE) {
					const int r = r0 + lane / PIECES, piece = lane % PIECES, n = n0 + 4 * piece;
					v4f v = scratch[r * PIECES + (piece ^ (r % PIECES))];
					if (m + r < M && n < N) {
						const int64_t at = static_cast<int64_t>(m + r) * N + n;
						value out[4];
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
					}
				}
			} else {
				constexpr int LANES = 16 * FN < 64 ? 16 * FN : 64, AT_ONCE = 64 / LANES;
#pragma unroll
				for (int r0 = 0; r0 < 16; r0 += AT_ONCE) {
					const int r = r0 + lane / LANES;
#pragma unroll
					for (int c = lane % LANES; c < 16 * FN; c += LANES) {
						float v = scratch[r * PIECES + ((c >> 2) ^ (r % PIECES))][c & 3];
						if (m + r < M && n0 + c < N) {
							const int64_t at = static_cast<int64_t>(m + r) * N + n0 + c;
							y[at]			 = T::narrow(residual ? v + T::widen(residual[at]) : v);
						}
					}
				}
			}
			__builtin_amdgcn_wave_barrier();
		}
	}
};

template<int TYPE> hipError_t gemm(const i8_matrix& w, const i8_matrix& x, const void* residual, void* y, hipStream_t stream) {
	typedef typename i8_type<TYPE>::store value;
	const i8_store<TYPE> epi{ static_cast<value*>(y), static_cast<const value*>(residual), x.rows, w.rows };
	i8_launch_product<false>(i8_form_for(w.strips, x.strips, w.steps), w, x, 0, w.rows, epi, stream);
	return hipGetLastError();
}

} // namespace

hipError_t launch_i8_gemm(const i8_matrix& w, const i8_matrix& x, const void* residual, void* y, int type, hipStream_t stream) {
	return type == NH_F32 ? gemm<NH_F32>(w, x, residual, y, stream) : type == NH_F16 ? gemm<NH_F16>(w, x, residual, y, stream) : gemm<NH_BF16>(w, x, residual, y, stream);
}

} // namespace nh
