// y [M][N] = x . w^T (+ residual) for int8 matrices with a scale per row, gfx950:  y[m][n] = sx[m] sw[n] sum_k x[m][k] w[n][k]
//
// The sums are whole numbers and exact (K is limited so that they stay below 2^31); each is brought to fp32, scaled by the row's and then by the channel's scale, the residual added,
// and rounded once to y's type.  The kernels are in i8_product.h.
#include "i8_product.h"
#include "i8_values.h"

namespace nh {

namespace {

template<int TYPE> struct i8_store {
	typedef i8_type<TYPE> T;
	typedef typename T::store value;
	value* y;
	const value* residual;
	int M, N;

	// the only row's sums of a strip of n, in all of a fragment's columns
	__device__ __forceinline__ void token(v4i sums, int n0, float sx, const i8_matrix& w) const {
		const int lane = threadIdx.x & 63, n = n0 + 4 * (lane >> 4) + (lane & 3);
		if ((lane & 15) < 4 && n < N) { // a lane takes one of its four
			const int sum = (lane & 2) ? (lane & 1) ? sums[3] : sums[2] : (lane & 1) ? sums[1] : sums[0];
			const float v = static_cast<float>(sum) * sx * w.scale[n];
			y[n]		  = T::narrow(residual ? v + T::widen(residual[n]) : v);
		}
	}

	// A lane has four neighbouring n of sixteen different rows m: sixteen rows at a time go through LDS, so that a wave's loads and stores run along the rows, four values to a lane.  Pieces of four
	// values lie at places permuted by the row, which spreads them over the banks either way.  The residual of the next sixteen rows is on its way while these are stored (y may be the residual: a
	// row's is loaded before any of that row is stored).  FOURS: N is a multiple of four.  If not, a row's fours lie at any multiple of a value's size, which the card's loads and stores take, and its
	// last values go one by one.
	template<int FN, int FM, bool FOURS> __device__ __forceinline__ void along_rows(const v4i (&sums)[FN][FM], int n0, int m0, const i8_matrix& w, const i8_matrix& x, v4f* scratch) const {
		constexpr int PIECES = 4 * FN, LANES = PIECES < 64 ? PIECES : 64, ROWS = 64 / LANES, TIMES = 16 / ROWS;
		const int lane = threadIdx.x & 63, row = lane & 15;
		const int c0 = lane % LANES, r0 = lane / LANES, n = n0 + 4 * c0; // this lane's piece and first row when it moves values
		struct values {
			value v[4];
		};
		constexpr int ALIGNMENT = FOURS ? sizeof(values) : sizeof(value);
		const bool four			= FOURS || n + 4 <= N;
		constexpr int SETS = FN < 8 ? 2 : 1; // (in the largest tiles the sums leave no room for two)
		values add[SETS][TIMES] = {};
		auto fetch = [&](int i, values(&to)[TIMES]) { // (past the end: the last ones, for nothing)
#pragma unroll
			for (int t = 0; t < TIMES; ++t) {
				const value* from = residual + static_cast<int64_t>(min(m0 + 16 * i + r0 + ROWS * t, M - 1)) * N;
				if (four) {
					__builtin_memcpy(&to[t], __builtin_assume_aligned(from + (FOURS ? min(n, N - 4) : n), ALIGNMENT), sizeof(values));
				} else {
#pragma unroll
					for (int e = 0; e < 4; ++e) {
						to[t].v[e] = from[min(n + e, N - 1)];
					}
				}
			}
		};
		// all scales before the first store: a wait for a load is also one for the stores before it
		v4f sw[FN];
		float sx[FM];
#pragma unroll
		for (int f = 0; f < FN; ++f) {
			sw[f] = i8_scales4(w, n0 + 4 * (4 * f + (lane >> 4)));
		}
#pragma unroll
		for (int i = 0; i < FM; ++i) {
			const int m = m0 + 16 * i + row;
			sx[i]		= m < M ? x.scale[m] : 0.0f;
		}
		if (residual && SETS == 2) {
			fetch(0, add[0]);
		}
#pragma unroll
		for (int i = 0; i < FM; ++i) {
			if (residual && SETS == 1) {
				fetch(i, add[0]);
			}
			const int m = m0 + 16 * i;
#pragma unroll
			for (int f = 0; f < FN; ++f) {
				const int piece = 4 * f + (lane >> 4);
				v4f v;
#pragma unroll
				for (int e = 0; e < 4; ++e) {
					v[e] = static_cast<float>(sums[f][i][e]) * sx[i] * sw[f][e];
				}
				scratch[row * PIECES + (piece ^ (row % PIECES))] = v;
			}
			if (residual && SETS == 2 && i + 1 < FM) {
				fetch(i + 1, add[(i + 1) % SETS]);
			}
			__builtin_amdgcn_wave_barrier(); // (one wave's own LDS accesses are in order)
#pragma unroll
			for (int t = 0; t < TIMES; ++t) {
				const int r = r0 + ROWS * t;
				const v4f v = scratch[r * PIECES + (c0 ^ (r % PIECES))];
				values out;
#pragma unroll
				for (int e = 0; e < 4; ++e) {
					out.v[e] = T::narrow(residual ? v[e] + T::widen(add[i % SETS][t].v[e]) : v[e]);
				}
				value* to = y + static_cast<int64_t>(m + r) * N + n;
				if (m + r < M && four && n < N) {
					__builtin_memcpy(__builtin_assume_aligned(to, ALIGNMENT), &out, sizeof(values));
				} else if (!FOURS && m + r < M) {
#pragma unroll
					for (int e = 0; e < 4; ++e) {
						if (n + e < N) {
							to[e] = out.v[e];
						}
					}
				}
			}
			__builtin_amdgcn_wave_barrier();
		}
	}
	template<int FN, int FM> __device__ __forceinline__ void operator()(const v4i (&sums)[FN][FM], int n0, int m0, const i8_matrix& w, const i8_matrix& x, v4f* scratch) const {
		if ((N & 3) == 0) {
			along_rows<FN, FM, true>(sums, n0, m0, w, x, scratch);
		} else {
			along_rows<FN, FM, false>(sums, n0, m0, w, x, scratch);
		}
	}
};

// Up to ROWS rows, quantized inside (behind the norm if there is one): every workgroup brings the rows to 8 bits in LDS by itself, which takes less than a launch of its own and the wait for it, while
// the first of its weights are on their way.  Then as i8_rows_product for one strip of x, whose other rows repeat the last one.  PIECES: of eight values per thread, so K up to 4096 PIECES.
template<int TYPE, bool NORM, int ROWS, int PIECES, int FN> __global__ __launch_bounds__(512) void i8_token_product(i8_matrix w, const void* x, const float* norm, double part, float eps, int K, int64_t stride, int n_tiles,
	i8_store<TYPE> epi) {
	constexpr int WAVES = 8, AHEAD = 8 / FN;
	__shared__ v4u row[PIECES * 256 * ROWS]; // [step][16 values][row]
	__shared__ v4i parts[WAVES][FN][64];
	__shared__ double squares[ROWS][WAVES];
	__shared__ uint32_t tops[ROWS][WAVES];
	__shared__ float scales[I8_ROWS];
	const i8_place p = i8_place_of(n_tiles, 1);
	if (!p.there) {
		return;
	}
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	const int pieces = 8 * w.steps;
	float v[ROWS][PIECES][8];
#pragma unroll
	for (int i = 0; i < ROWS; ++i) {
#pragma unroll
		for (int j = 0; j < PIECES; ++j) {
			const int c = threadIdx.x + 512 * j;
			if (c < pieces) {
				i8_load<TYPE>(x, min(i, epi.M - 1) * stride + 8 * c, K - 8 * c, v[i][j]);
			}
		}
	}
	const int n_strip = p.n * FN;
	const v4u* a[FN];
#pragma unroll
	for (int f = 0; f < FN; ++f) {
		a[f] = w.q + static_cast<int64_t>(min(n_strip + f, w.strips - 1)) * w.steps * 64 + lane;
	}
	const int per = (w.steps + WAVES - 1) / WAVES, begin = wave * per, end = min(w.steps, begin + per), last = max(min(end, w.steps) - 1, 0);
	v4u ahead[AHEAD][FN];
	auto load = [&](int s) { // (past the wave's last step: that one again, or any where it has none)
#pragma unroll
		for (int u = 0; u < AHEAD; ++u) {
#pragma unroll
			for (int f = 0; f < FN; ++f) {
				ahead[u][f] = a[f][min(s + u, last) * 64];
			}
		}
	};
	load(begin);
	if constexpr (NORM) {
		double sum[ROWS] = {};
#pragma unroll
		for (int i = 0; i < ROWS; ++i) {
#pragma unroll
			for (int j = 0; j < PIECES; ++j) {
				if (threadIdx.x + 512 * j < static_cast<unsigned>(pieces)) {
#pragma unroll
					for (int e = 0; e < 8; ++e) {
						sum[i] = fma(static_cast<double>(v[i][j][e]), static_cast<double>(v[i][j][e]), sum[i]);
					}
				}
			}
#pragma unroll
			for (int d = 32; d > 0; d >>= 1) {
				sum[i] += __shfl_xor(sum[i], d);
			}
			if (lane == 0) {
				squares[i][wave] = sum[i];
			}
		}
		__syncthreads();
		float r[ROWS];
#pragma unroll
		for (int i = 0; i < ROWS; ++i) {
			sum[i] = squares[i][0];
#pragma unroll
			for (int u = 1; u < WAVES; ++u) {
				sum[i] += squares[i][u];
			}
			r[i] = i8_rms(sum[i], part, eps);
		}
#pragma unroll
		for (int j = 0; j < PIECES; ++j) {
			const int c = threadIdx.x + 512 * j;
			if (c < pieces) {
				float g[8];
				i8_load<NH_F32>(norm, 8 * c, K - 8 * c, g);
#pragma unroll
				for (int i = 0; i < ROWS; ++i) {
#pragma unroll
					for (int e = 0; e < 8; ++e) {
						v[i][j][e] = __fmul_rn(__fmul_rn(v[i][j][e], r[i]), g[e]);
					}
				}
			}
		}
	}
#pragma unroll
	for (int i = 0; i < ROWS; ++i) {
		uint32_t top = 0;
#pragma unroll
		for (int j = 0; j < PIECES; ++j) {
			if (threadIdx.x + 512 * j < static_cast<unsigned>(pieces)) {
#pragma unroll
				for (int e = 0; e < 8; ++e) {
					top = max(top, __float_as_uint(v[i][j][e]) & 0x7FFFFFFFu);
				}
			}
		}
#pragma unroll
		for (int d = 32; d > 0; d >>= 1) {
			top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), d)));
		}
		if (lane == 0) {
			tops[i][wave] = top;
		}
	}
	__syncthreads();
	float scale = 0.0f; // of the only row
#pragma unroll
	for (int i = 0; i < ROWS; ++i) {
		uint32_t top = tops[i][0];
#pragma unroll
		for (int u = 1; u < WAVES; ++u) {
			top = max(top, tops[i][u]);
		}
		const i8_step step(top);
		scale = step.scale;
		if (ROWS > 1 && threadIdx.x == 0) {
			scales[i] = scale;
		}
#pragma unroll
		for (int j = 0; j < PIECES; ++j) {
			const int c = threadIdx.x + 512 * j;
			if (c < pieces) {
				uint32_t out[2];
				step.round(v[i][j], out);
				reinterpret_cast<v2u*>(row)[((c >> 1) * ROWS + i) * 2 + (c & 1)] = v2u{ out[0], out[1] };
			}
		}
	}
	__syncthreads();
	v4i sums[FN][1] = {};
	const v4u* b = row + (lane >> 4) * ROWS + min(lane & 15, ROWS - 1);
#pragma unroll 1
	for (int s = begin; s < end;) {
#pragma unroll
		for (int u = 0; u < AHEAD; ++u) {
			if (s + u < end) {
#pragma unroll
				for (int f = 0; f < FN; ++f) {
					sums[f][0] = i8_mfma(ahead[u][f], b[4 * ROWS * (s + u)], sums[f][0]);
				}
			}
		}
		s += AHEAD;
		if (s < end) {
			load(s);
		}
	}
#pragma unroll
	for (int f = 0; f < FN; ++f) {
		parts[wave][f][lane] = sums[f][0];
	}
	__syncthreads();
	if (wave < FN) {
		v4i all = parts[0][wave][lane];
#pragma unroll
		for (int i = 1; i < WAVES; ++i) {
			all += parts[i][wave][lane];
		}
		if constexpr (ROWS == 1) {
			epi.token(all, (n_strip + wave) * I8_ROWS, scale, w);
		} else {
			const v4i only[1][1] = { { all } };
			const i8_matrix there{ nullptr, scales, epi.M, 1, w.steps };
			epi.template operator()<1, 1>(only, (n_strip + wave) * I8_ROWS, 0, w, there, reinterpret_cast<v4f*>(&parts[0][wave][0]));
		}
	}
}

// ns that a byte of 16 x 16 results takes (i8_form_for)
constexpr int64_t STORE = 39;

template<int TYPE> hipError_t gemm(const i8_matrix& w, const i8_matrix& x, const void* residual, void* y, hipStream_t stream) {
	typedef typename i8_type<TYPE>::store value;
	const i8_store<TYPE> epi{ static_cast<value*>(y), static_cast<const value*>(residual), x.rows, w.rows };
	i8_launch_product<false>(i8_form_for(w.strips, x.strips, w.steps, STORE * int64_t{ sizeof(value) }), w, x, 0, w.rows, epi, stream);
	return hipGetLastError();
}

template<int TYPE, bool NORM> hipError_t token(const i8_matrix& w, const i8_rows& in, const void* residual, void* y, hipStream_t stream) {
	typedef typename i8_type<TYPE>::store value;
	const i8_store<TYPE> epi{ static_cast<value*>(y), static_cast<const value*>(residual), in.rows, w.rows };
	auto launch = [&](auto kernel, int n_strips) {
		const int n_tiles = (w.strips + n_strips - 1) / n_strips;
		kernel<<<i8_grid(n_tiles, 1), 512, 0, stream>>>(w, in.x, in.norm, in.part, in.eps, in.k, in.stride, n_tiles, epi);
	};
	const bool few = w.strips <= 512; // so that there are workgroups for all CUs
	if (in.rows > 2) {
		if constexpr (!NORM) {
			few ? launch(i8_token_product<TYPE, false, 4, 1, 1>, 1) : launch(i8_token_product<TYPE, false, 4, 1, 2>, 2);
		}
	} else if (in.rows == 2) {
		few ? launch(i8_token_product<TYPE, NORM, 2, 2, 1>, 1) : launch(i8_token_product<TYPE, NORM, 2, 2, 2>, 2);
	} else if (w.steps <= 64) {
		few ? launch(i8_token_product<TYPE, NORM, 1, 1, 1>, 1) : launch(i8_token_product<TYPE, NORM, 1, 1, 2>, 2);
	} else {
		few ? launch(i8_token_product<TYPE, NORM, 1, 4, 1>, 1) : launch(i8_token_product<TYPE, NORM, 1, 4, 2>, 2);
	}
	return hipGetLastError();
}
template<int TYPE> hipError_t token(const i8_matrix& w, const i8_rows& in, const void* residual, void* y, hipStream_t stream) {
	return in.norm ? token<TYPE, true>(w, in, residual, y, stream) : token<TYPE, false>(w, in, residual, y, stream);
}

} // namespace

// Measured, us as here / as two launches, fp32: one row of 4096 against 1024 rows of w 3.5 / 6.4, 4096 5.0 / 8.2, 14336 10.8 / 13.9, 128256 83 / 83; two rows 4096 6.7 / 8.3, 32768 25.8 / 29.4, 65536 47.7 / 48.7, behind
// a norm 50.5 / 50; four rows 4096 7.6 / 8.4, 14336 11.6 / 14.0, 32768 28.8 / 29.6, 65536 52 / 49, behind a norm 4096 9.6 / 9.3.
bool i8_token_fits(int64_t m, int64_t n, int64_t k, bool norm) {
	return (m == 1 && k <= 16384) || (n <= 32768 && ((m == 2 && k <= 8192) || (m > 2 && m <= 4 && k <= 4096 && !norm)));
}
hipError_t launch_i8_token(const i8_matrix& w, const i8_rows& in, int type, const void* residual, void* y, hipStream_t stream) {
	return type == NH_F32 ? token<NH_F32>(w, in, residual, y, stream) : type == NH_F16 ? token<NH_F16>(w, in, residual, y, stream) : token<NH_BF16>(w, in, residual, y, stream);
}

hipError_t launch_i8_gemm(const i8_matrix& w, const i8_matrix& x, const void* residual, void* y, int type, hipStream_t stream) {
	return type == NH_F32 ? gemm<NH_F32>(w, x, residual, y, stream) : type == NH_F16 ? gemm<NH_F16>(w, x, residual, y, stream) : gemm<NH_BF16>(w, x, residual, y, stream);
}

} // namespace nh
