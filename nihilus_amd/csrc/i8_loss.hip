// Softmax cross entropy of rows on a vocabulary projection in int8 with a scale per row, and its gradient, gfx950.  No logits are kept.
//
//   l[m][n] = sx[m] sw[n] sum_k x[m][k] w[n][k],   lse[m] = log sum_n exp l[m][n],   loss[m] = lse[m] - l[m][t[m]]
//
// Forward: the product kernels of i8_product.h with an epilogue that leaves of each stretch of a row's logits its maximum and the sum of exp(l - maximum), and the target's logit where
// it comes by; a second kernel joins the stretches.
//
// Backward: dx[m][k] = grad[m] sum_n d[m][n] sw[n] w[n][k],  d = exp(l - lse) - [n = t].  Pieces of the vocabulary at a time, the product kernels form l again and leave
// P = d sw 2^e in fp16, in operand order; a second product sums P w over n.  d is at most 1 - exp(-loss) of its row, so e is chosen by the row (and by the largest of all sw): P is below 2^14, and what
// is 2^-28 of the row's largest is still a normal number.  fp16 has 11 bits; where dx is fp32, P is a sum of two such numbers (22 bits) and the second product twice as much.
// w enters the second product as fp16, exactly.  It lies in fragments of 16 rows n x 64 values k, and the sum is over n: ds_read_b64_tr_b8 takes eight rows of sixteen columns out of LDS so that
// a lane has eight n of one k.
#include "i8_product.h"

#include <algorithm>

namespace nh {

namespace {

constexpr float LOG2_E = 1.44269504088896340736f;

// 2^x, within 2 ulp for the arguments here (x <= 0 up to rounding)
__device__ __forceinline__ float exp2_native(float x) {
	return __builtin_amdgcn_exp2f(x);
}

// part: [stretch][M] (maximum, sum below it)
struct i8_stretches {
	float2* parts;
	float* hit; // [M] the target's logit
	const int32_t* targets;
	int M, N;

	template<int FN, int FM> __device__ __forceinline__ void operator()(const v4i (&sums)[FN][FM], int n0, int m0, const i8_matrix& w, const i8_matrix& x, v4f*) const {
		const int lane = threadIdx.x & 63;
		if (n0 >= N) {
			return;
		}
#pragma unroll
		for (int i = 0; i < FM; ++i) {
			const int m		 = m0 + 16 * i + (lane & 15);
			const bool there = m < M;
			const float sx	 = there ? x.scale[m] : 0.0f;
			const int target = there ? targets[m] : -1;
			float top		 = -__builtin_inff();
#pragma unroll
			for (int f = 0; f < FN; ++f) {
				const int n	 = n0 + 16 * f + 4 * (lane >> 4);
				const v4f sw = i8_scales4(w, n);
#pragma unroll
				for (int e = 0; e < 4; ++e) {
					const float l = static_cast<float>(sums[f][i][e]) * sx * sw[e];
					top			  = n + e < N ? fmaxf(top, l) : top;
					if (n + e == target && n + e < N) {
						hit[m] = l;
					}
				}
			}
			top = fmaxf(top, __shfl_xor(top, 16));
			top = fmaxf(top, __shfl_xor(top, 32));
			float sum = 0.0f;
#pragma unroll
			for (int f = 0; f < FN; ++f) {
				const int n	 = n0 + 16 * f + 4 * (lane >> 4);
				const v4f sw = i8_scales4(w, n);
#pragma unroll
				for (int e = 0; e < 4; ++e) {
					const float l = static_cast<float>(sums[f][i][e]) * sx * sw[e];
					sum += n + e < N ? exp2_native((l - top) * LOG2_E) : 0.0f;
				}
			}
			sum += __shfl_xor(sum, 16);
			sum += __shfl_xor(sum, 32);
			if (there && lane < 16) {
				parts[static_cast<int64_t>(n0 / (16 * FN)) * M + m] = make_float2(top, sum);
			}
		}
	}
};

// 16 rows to a workgroup, 64 threads to a row
__global__ __launch_bounds__(1024) void i8_join_stretches(const float2* parts, const float* hit, const int32_t* targets, float* losses, float* lse, int M, int N, int count) {
	__shared__ float2 all[64][16];
	const int col = threadIdx.x & 15, lane = threadIdx.x >> 4, m = blockIdx.x * 16 + col;
	float top = -__builtin_inff(), sum = 0.0f;
	if (m < M) {
		for (int i = lane; i < count; i += 64) {
			const float2 p	= parts[static_cast<int64_t>(i) * M + m];
			const float now = fmaxf(top, p.x);
			// (a stretch whose logits are all NaN has -infinity and NaN)
			sum = (top == now ? sum : sum * exp2_native((top - now) * LOG2_E)) + (p.x == now ? p.y : p.y * exp2_native((p.x - now) * LOG2_E));
			top = now;
		}
	}
	all[lane][col] = make_float2(top, sum);
	__syncthreads();
	if (threadIdx.x < 16 && m < M) {
		for (int i = 0; i < 64; ++i) {
			top = fmaxf(top, all[i][col].x);
		}
		sum = 0.0f;
		for (int i = 0; i < 64; ++i) {
			const float2 p = all[i][col];
			sum += p.x == top ? p.y : p.y * exp2_native((p.x - top) * LOG2_E);
		}
		const float l = top + logf(sum);
		lse[m]		  = l;
		losses[m]	  = targets[m] >= 0 && targets[m] < N ? l - hit[m] : 0.0f;
	}
}

constexpr int64_t up(int64_t n, int64_t to) {
	return (n + to - 1) / to * to;
}

// ---- backward ----

constexpr int MAXIMA = 64;
__global__ __launch_bounds__(256) void i8_largest_scales(const float* scale, int n, float* out) {
	__shared__ float tops[4];
	float top = 0.0f;
	for (int i = blockIdx.x * 256 + threadIdx.x; i < n; i += MAXIMA * 256) {
		top = fmaxf(top, fabsf(scale[i]));
	}
#pragma unroll
	for (int d = 32; d > 0; d >>= 1) {
		top = fmaxf(top, __shfl_xor(top, d));
	}
	if ((threadIdx.x & 63) == 0) {
		tops[threadIdx.x >> 6] = top;
	}
	__syncthreads();
	if (threadIdx.x == 0) {
		out[blockIdx.x] = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
	}
}
// f, such that the largest scale times 2^f is in [1/2, 1) (any f if it is 0 or not finite)
__device__ __forceinline__ int scales_exponent(const float* maxima) {
	float top = maxima[threadIdx.x & 63];
#pragma unroll
	for (int d = 32; d > 0; d >>= 1) {
		top = fmaxf(top, __shfl_xor(top, d));
	}
	int e = 0;
	if (top > 0.0f && top < __builtin_inff()) {
		(void)frexpf(top, &e);
	}
	return -e;
}
// e, such that 2^e (1 - exp(-loss)) is in [2^12, 2^13); where that is below 2^-16, lse itself does not tell such d from nothing
__device__ __forceinline__ int slopes_exponent(float loss) {
	const float most = fminf(fmaxf(1.0f - exp2_native(-loss * LOG2_E), 0x1p-16f), 1.0f);
	int e;
	(void)frexpf(most, &e);
	return 13 - e;
}

// P of a piece of the vocabulary: [term][strip of 16 rows][32 n][lane], lane's eight numbers n = 16 h + 4 (lane / 16) + i at 4 h + i, row lane % 16
template<int TERMS> struct i8_slopes {
	v8h* p;
	const int32_t* targets;
	const float *losses, *lse, *maxima;
	int M, N, first_n, blocks; // of 32 n in the piece

	template<int FN, int FM> __device__ __forceinline__ void operator()(const v4i (&sums)[FN][FM], int n0, int m0, const i8_matrix& w, const i8_matrix& x, v4f*) const {
		static_assert(FN % 2 == 0);
		const int lane = threadIdx.x & 63, block = (n0 - first_n) / 32;
		const int f	   = scales_exponent(maxima);
#pragma unroll
		for (int i = 0; i < FM; ++i) {
			const int strip = m0 / 16 + i, m = 16 * strip + (lane & 15);
			if (strip >= x.strips) {
				continue;
			}
			const int target  = m < M ? targets[m] : -1;
			const bool scored = target >= 0 && target < N;
			const float sx = scored ? x.scale[m] : 0.0f, below = scored ? lse[m] : 0.0f;
			const float lift = scored ? ldexpf(1.0f, slopes_exponent(losses[m])) : 0.0f;
#pragma unroll
			for (int b = 0; b < FN / 2; ++b) {
				if (block + b >= blocks) {
					continue;
				}
				v8h out[TERMS];
#pragma unroll
				for (int h = 0; h < 2; ++h) {
					const int n	 = n0 + 32 * b + 16 * h + 4 * (lane >> 4);
					const v4f sw = i8_scales4(w, n);
#pragma unroll
					for (int e = 0; e < 4; ++e) {
						const float l = static_cast<float>(sums[2 * b + h][i][e]) * sx * sw[e];
						const float d = exp2_native((l - below) * LOG2_E) - (n + e == target ? 1.0f : 0.0f);
						float v		  = scored && n + e < N ? d * lift * ldexpf(sw[e], f) : 0.0f;
#pragma unroll
						for (int t = 0; t < TERMS; ++t) {
							out[t][4 * h + e] = static_cast<_Float16>(v);
							v -= static_cast<float>(out[t][4 * h + e]);
						}
					}
				}
#pragma unroll
				for (int t = 0; t < TERMS; ++t) {
					p[((static_cast<int64_t>(t) * x.strips + strip) * blocks + block + b) * 64 + lane] = out[t];
				}
			}
		}
	}
};

// Eight rows n (of 32, two fragments of 16 x 64 beside each other in LDS) of column k as fp16, for the lane's place in the A operand of v_mfma_f32_16x16x32_f16: columns 16 c + lane % 16 of the
// fragments, rows 4 (lane / 16) + i of the first and of the second.  In a group of sixteen lanes lane 2 j + h names row j, columns 8 h .. 8 h + 7 of sixteen, and lane L gets column L of all eight rows.
typedef int v2i __attribute__((ext_vector_type(2)));
__device__ __forceinline__ v8h i8_columns(const v4u* first, const v4u* second, int c, int lane) {
	const int j = (lane & 15) >> 1, row = 4 * (lane >> 4) + (j & 3);
	const char* at = reinterpret_cast<const char*>(j < 4 ? first : second) + (c * 16 + row) * 16 + 8 * (lane & 1);
	const v2i raw  = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) v2i*)(const_cast<char*>(at)));
	v8h out;
#pragma unroll
	for (int d = 0; d < 2; ++d) {
		// 128 + q as the low byte of 0x6400 + ... is the fp16 number 1024 + 128 + q
		const uint32_t u = static_cast<uint32_t>(raw[d]) ^ 0x80808080u;
		const v2h low = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)), high = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u));
		const v2h a = low - static_cast<_Float16>(1152.0f), b = high - static_cast<_Float16>(1152.0f);
		out[4 * d] = a[0], out[4 * d + 1] = a[1], out[4 * d + 2] = b[0], out[4 * d + 3] = b[1];
	}
	return out;
}

struct i8_slope_product {
	const v8h* p; // as i8_slopes leaves it
	float* out; // [split][M][columns]
	int M, columns, strips, blocks, first_block; // columns: 64 w.steps; first_block: of the vocabulary, in 32 n
	int per; // blocks of a split
	bool add;
};

// A workgroup has 16 WK FK columns x 16 WM FM rows of sums over its split's blocks of 32 n, in a ring as the product kernel for many rows.
template<int WK, int WM, int FK, int FM, int TERMS, int RING> __global__ __launch_bounds__(64 * WK * WM, 2) void i8_slope_kernel(i8_matrix w, i8_slope_product a, int k_tiles, int m_tiles) {
	constexpr int WAVES = WK * WM, STEPS = WK * FK / 4, NF = 2 * STEPS, FRAGMENTS = NF + WM * FM * TERMS, LOADS = (FRAGMENTS + WAVES - 1) / WAVES;
	static_assert(WK * FK % 4 == 0);
	__shared__ v4u ring[RING][FRAGMENTS][64];
	const int split = blockIdx.y;
	const i8_place p = i8_place_of(k_tiles, m_tiles);
	if (!p.there) {
		return;
	}
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wk = wave % WK, wm = wave / WK;
	const int step0 = p.n * STEPS, strip0 = p.m * WM * FM;
	const int begin = split * a.per, blocks = min(a.per, a.blocks - begin);
	auto load = [&](int s) {
		const int block = begin + s;
#pragma unroll
		for (int j = 0; j < LOADS; ++j) { // (past the last fragment: that one again, to the same place)
			const int f = min(wave * LOADS + j, FRAGMENTS - 1);
			const v4u* from;
			if (f < NF) { // fragments [step][2]
				from = w.q + (static_cast<int64_t>(min(2 * (a.first_block + block) + (f & 1), w.strips - 1)) * w.steps + min(step0 + (f >> 1), w.steps - 1)) * 64;
			} else {
				const int t = (f - NF) % TERMS, strip = min(strip0 + (f - NF) / TERMS, a.strips - 1);
				from		= reinterpret_cast<const v4u*>(a.p) + ((static_cast<int64_t>(t) * a.strips + strip) * a.blocks + block) * 64;
			}
			load_global_to_lds_b128(from, 16 * lane, &ring[s % RING][f][0]);
		}
	};
	auto arrive = [&](int s, int asked) { // step s is in LDS, steps below `asked` may be on their way
		const int ahead = min(blocks, asked) - 1 - s;
		if (ahead >= 2) {
			i8_arrive<2 * LOADS>();
		} else if (ahead == 1) {
			i8_arrive<LOADS>();
		} else {
			i8_arrive<0>();
		}
	};
	v4f sums[FK][FM] = {};
	for (int s = 0; s < min(blocks, RING - 1); ++s) {
		load(s);
	}
	for (int s = 0; s < blocks; ++s) {
		arrive(s, s + RING - 1); // (and everybody has read the step before)
		if (s + RING - 1 < blocks) {
			load(s + RING - 1);
		}
		const auto& at = ring[s % RING];
		v8h k[FK];
#pragma unroll
		for (int f = 0; f < FK; ++f) {
			const int c = wk * FK + f;
			k[f]		= i8_columns(at[2 * (c >> 2)], at[2 * (c >> 2) + 1], c & 3, lane);
		}
#pragma unroll
		for (int i = 0; i < FM; ++i) {
#pragma unroll
			for (int t = TERMS - 1; t >= 0; --t) { // the small term first
				const v8h d = __builtin_bit_cast(v8h, at[NF + (wm * FM + i) * TERMS + t][lane]);
#pragma unroll
				for (int f = 0; f < FK; ++f) {
					sums[f][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[f], d, sums[f][i], 0, 0, 0);
				}
			}
		}
	}
#pragma unroll
	for (int i = 0; i < FM; ++i) {
		const int m = 16 * (strip0 + wm * FM + i) + (lane & 15);
		if (m >= a.M) {
			continue;
		}
#pragma unroll
		for (int f = 0; f < FK; ++f) {
			const int k = 64 * step0 + 16 * (wk * FK + f) + 4 * (lane >> 4);
			if (k < a.columns) {
				v4f* to = reinterpret_cast<v4f*>(a.out + (static_cast<int64_t>(split) * a.M + m) * a.columns + k);
				*to		= a.add ? *to + sums[f][i] : sums[f][i];
			}
		}
	}
}

// the splits' sums, brought back from the powers of two, times the row's grad
template<int TYPE> __global__ __launch_bounds__(256) void i8_slope_results(const float* sums, const float* maxima, const int32_t* targets, const float* losses, const float* grad,
	typename i8_type<TYPE>::store* dx, int M, int N, int K, int columns, int splits) {
	const int f = scales_exponent(maxima);
	const int m = blockIdx.y * gridDim.z + blockIdx.z, k = 4 * (blockIdx.x * 256 + threadIdx.x);
	if (m >= M || k >= K) {
		return;
	}
	const bool scored = targets[m] >= 0 && targets[m] < N;
	v4f all{};
	for (int s = 0; s < splits; ++s) {
		all += *reinterpret_cast<const v4f*>(sums + (static_cast<int64_t>(s) * M + m) * columns + k);
	}
	const int back	= scored ? -f - slopes_exponent(losses[m]) : 0;
	const float g	= grad ? grad[m] : 1.0f;
#pragma unroll
	for (int e = 0; e < 4; ++e) {
		if (k + e < K) {
			dx[static_cast<int64_t>(m) * K + k + e] = i8_type<TYPE>::narrow(scored ? ldexpf(all[e], back) * g : 0.0f);
		}
	}
}

// How the backward pass is cut: pieces of the vocabulary by memory, splits of a piece so that the second product has some 256 workgroups.
struct gradient_plan {
	int64_t piece, blocks; // n, blocks of 32 n
	int64_t k_tiles, m_tiles, splits;
	int64_t slopes, sums; // bytes
	bool many;
	int terms;
};
gradient_plan plan_gradient(int64_t m, int64_t n, int64_t k, int type) {
	gradient_plan g{};
	const int64_t strips = i8_strips(m), steps = i8_steps(k);
	g.terms				 = type == NH_F32 ? 2 : 1;
	const int64_t row	 = strips * 16 * 2 * g.terms;
	g.piece				 = std::min(up(n, 32), std::max<int64_t>((int64_t{ 1 } << 27) / row / 256 * 256, 1024));
	g.blocks			 = g.piece / 32;
	g.many				 = m > 64;
	g.k_tiles			 = (steps + 3) / 4;
	g.m_tiles			 = g.many ? (m + 255) / 256 : (m + 63) / 64;
	g.splits			 = std::max<int64_t>(1, std::min(g.blocks / 8, 256 / (g.k_tiles * g.m_tiles)));
	g.slopes			 = up(row * g.piece, 256);
	g.sums				 = up(g.splits * m * steps * I8_STEP * 4, 256);
	return g;
}

template<int TERMS> void gradient_sums(const i8_matrix& w, const i8_matrix& x, const i8_gradient& g, const gradient_plan& plan, v8h* slopes, float* sums, const float* maxima, hipStream_t stream) {
	for (int64_t first = 0; first < w.rows; first += plan.piece) {
		const int64_t n = std::min<int64_t>(plan.piece, w.rows - first), blocks = (n + 31) / 32;
		const i8_slopes<TERMS> epi{ slopes, g.targets, g.losses, g.lse, maxima, x.rows, w.rows, static_cast<int>(first), static_cast<int>(blocks) };
		i8_launch_product<true>(i8_form_for(i8_strips(n), x.strips, w.steps), w, x, static_cast<int>(first), static_cast<int>(n), epi, stream);
		i8_slope_product a{};
		a.p = slopes, a.out = sums;
		a.M = x.rows, a.columns = w.steps * I8_STEP, a.strips = x.strips, a.blocks = static_cast<int>(blocks), a.first_block = static_cast<int>(first / 32);
		a.per = static_cast<int>((blocks + plan.splits - 1) / plan.splits);
		a.add = first > 0;
		const dim3 grid(i8_grid(plan.k_tiles, plan.m_tiles), static_cast<unsigned>(plan.splits));
		if (plan.many) {
			i8_slope_kernel<4, 2, 4, 8, TERMS, TERMS == 1 ? 4 : 3><<<grid, 512, 0, stream>>>(w, a, static_cast<int>(plan.k_tiles), static_cast<int>(plan.m_tiles));
		} else {
			i8_slope_kernel<4, 2, 4, 2, TERMS, 4><<<grid, 512, 0, stream>>>(w, a, static_cast<int>(plan.k_tiles), static_cast<int>(plan.m_tiles));
		}
	}
}

} // namespace

// (K is not known here: room for the shortest stretches)
int64_t i8_losses_workspace(int64_t m, int64_t n) {
	return up(m * 4, 256) + up((n + 31) / 32 * m * 8, 256);
}

hipError_t launch_i8_losses(const i8_matrix& w, const i8_matrix& x, const i8_losses& l, hipStream_t stream) {
	char* ws		   = static_cast<char*>(l.workspace);
	float* hit		   = reinterpret_cast<float*>(ws);
	float2* parts	   = reinterpret_cast<float2*>(ws + up(static_cast<int64_t>(x.rows) * 4, 256));
	const i8_form form = i8_form_for(w.strips, x.strips, w.steps);
	const int each	   = i8_stretch(form);
	i8_launch_product<true>(form, w, x, 0, w.rows, i8_stretches{ parts, hit, l.targets, x.rows, w.rows }, stream);
	i8_join_stretches<<<(x.rows + 15) / 16, 1024, 0, stream>>>(parts, hit, l.targets, l.losses, l.lse, x.rows, w.rows, (w.rows + each - 1) / each);
	return hipGetLastError();
}

int64_t i8_gradient_workspace(int64_t m, int64_t n, int64_t k, int type) {
	const gradient_plan g = plan_gradient(m, n, k, type);
	return MAXIMA * 4 + g.slopes + g.sums;
}

hipError_t launch_i8_gradient(const i8_matrix& w, const i8_matrix& x, const i8_gradient& g, hipStream_t stream) {
	const gradient_plan plan = plan_gradient(x.rows, w.rows, g.k, g.type);
	char* ws				 = static_cast<char*>(g.workspace);
	float* maxima			 = reinterpret_cast<float*>(ws);
	v8h* slopes				 = reinterpret_cast<v8h*>(ws + MAXIMA * 4);
	float* sums				 = reinterpret_cast<float*>(ws + MAXIMA * 4 + plan.slopes);
	i8_largest_scales<<<MAXIMA, 256, 0, stream>>>(w.scale, w.rows, maxima);
	if (plan.terms == 2) {
		gradient_sums<2>(w, x, g, plan, slopes, sums, maxima, stream);
	} else {
		gradient_sums<1>(w, x, g, plan, slopes, sums, maxima, stream);
	}
	const int columns = w.steps * I8_STEP;
	const unsigned high = static_cast<unsigned>((x.rows + 63) / 64);
	const dim3 grid(static_cast<unsigned>((g.k + 1023) / 1024), high, 64);
	auto results = [&](auto kernel, auto* dx) {
		kernel<<<grid, 256, 0, stream>>>(sums, maxima, g.targets, g.losses, g.grad, dx, x.rows, w.rows, g.k, columns, static_cast<int>(plan.splits));
	};
	if (g.type == NH_F32) {
		results(i8_slope_results<NH_F32>, static_cast<float*>(g.dx));
	} else if (g.type == NH_F16) {
		results(i8_slope_results<NH_F16>, static_cast<uint16_t*>(g.dx));
	} else {
		results(i8_slope_results<NH_BF16>, static_cast<uint16_t*>(g.dx));
	}
	return hipGetLastError();
}

} // namespace nh
