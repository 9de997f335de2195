// Softmax cross entropy of rows on a vocabulary projection in int8 with a scale per row, and its gradient, gfx950.  No logits are kept.
//
//   l[m][n] = sx[m] sw[n] sum_k x[m][k] w[n][k],   lse[m] = log sum_n exp l[m][n],   loss[m] = lse[m] - l[m][t[m]]
//
// Forward: the product kernels of i8_product.h with an epilogue that leaves of each stretch of a row's logits its maximum and the sum of exp(l - maximum), and the target's logit where
// it comes by; a second kernel joins the stretches.
//
// Backward: dx[m][k] = grad[m] sum_n d[m][n] sw[n] w[n][k],  d = exp(l - lse) - [n = t].  Pieces of the vocabulary at a time, the product kernels form l again and leave
// P = d sw 2^e in fp16, in operand order; a second product sums P w over n.  d is at most 1 - exp(-loss) of its row, so e is chosen by the row (and by the largest of all sw): P is below 2^15, and what
// is 2^-28 of the row's largest is still a normal number.  P is a sum of two such numbers (22 bits), whatever dx is rounded to: with one (11 bits) 2048 rows of [128256 x 4096] took 2.6 ms instead of 3.7,
// and one bf16 dx in sixteen was another number.
// w enters the second product as fp16, exactly.  It lies in fragments of 16 rows n x 64 values k, and the sum is over n: ds_read_b64_tr_b8 takes eight rows of sixteen columns out of LDS so that
// a lane has eight n of one k.
#include "i8_product.h"

#include <algorithm>
#include <type_traits>

namespace nh {

namespace {

// ns that 16 x 16 exponentials take behind a product
constexpr int64_t EPILOGUE = 66;
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
		const int lane = threadIdx.x & 63, group = lane >> 4;
		if (n0 >= N) {
			return;
		}
		const bool all = n0 + 16 * FN <= N;
		v4f sw[FN];
#pragma unroll
		for (int f = 0; f < FN; ++f) {
			sw[f] = i8_scales4(w, n0 + 16 * f + 4 * group);
		}
		// all rows' before the first store: a wait for a load is also one for the stores before it
		float scales[FM];
		int places[FM];
#pragma unroll
		for (int i = 0; i < FM; ++i) {
			const int m	 = m0 + 16 * i + (lane & 15);
			scales[i]	 = m < M ? x.scale[m] : 0.0f;
			places[i]	 = m < M ? targets[m] : -1;
		}
#pragma unroll
		for (int i = 0; i < FM; ++i) {
			const int m		 = m0 + 16 * i + (lane & 15);
			const bool there = m < M;
			const float sx	 = scales[i];
			const int target = places[i];
			v4f l[FN];
			float top = -__builtin_inff();
#pragma unroll
			for (int f = 0; f < FN; ++f) {
#pragma unroll
				for (int e = 0; e < 4; ++e) {
					l[f][e] = static_cast<float>(sums[f][i][e]) * sx * sw[f][e];
				}
			}
			if (!all) { // nothing past the vocabulary
#pragma unroll
				for (int f = 0; f < FN; ++f) {
#pragma unroll
					for (int e = 0; e < 4; ++e) {
						l[f][e] = n0 + 16 * f + 4 * group + e < N ? l[f][e] : -__builtin_inff();
					}
				}
			}
			if (target >= n0 && target < n0 + 16 * FN && target < N) { // in this stretch
#pragma unroll
				for (int f = 0; f < FN; ++f) {
#pragma unroll
					for (int e = 0; e < 4; ++e) {
						if (n0 + 16 * f + 4 * group + e == target) {
							hit[m] = l[f][e];
						}
					}
				}
			}
#pragma unroll
			for (int f = 0; f < FN; ++f) {
				top = fmaxf(fmaxf(top, fmaxf(l[f][0], l[f][1])), fmaxf(l[f][2], l[f][3]));
			}
			top = fmaxf(top, __shfl_xor(top, 16));
			top = fmaxf(top, __shfl_xor(top, 32));
			// (an infinite largest one is not subtracted: a stretch of -infinities adds nothing, +infinity is the row's lse, and only NaN gives NaN)
			const float from = fabsf(top) < __builtin_inff() ? top : 0.0f;
			float sum		 = 0.0f;
#pragma unroll
			for (int f = 0; f < FN; ++f) {
#pragma unroll
				for (int e = 0; e < 4; ++e) {
					sum += exp2_native((l[f][e] - from) * LOG2_E);
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

// ROWS rows to a workgroup, neighbouring threads have neighbouring rows; joined among a wave's lanes first, then the waves', with one barrier (105 rows of [1088 x 1088] 6.9 us, 7.5 with a barrier a
// halving; few stretches: 128 threads to a row)
template<int ROWS, int THREADS> __global__ __launch_bounds__(THREADS) void i8_join_stretches(const float2* parts, const float* hit, const int32_t* targets, float* losses, float* lse, int M, int N, int count) {
	constexpr int LANES = THREADS / ROWS, AT_ONCE = 4, WAVES = THREADS / 64;
	__shared__ float2 all[WAVES][ROWS];
	const int col = threadIdx.x % ROWS, lane = threadIdx.x / ROWS, m = blockIdx.x * ROWS + col;
	const float none = -__builtin_inff();
	float top = none, sum = 0.0f;
	// (a stretch whose logits are all NaN has -infinity and NaN: equal maxima are not subtracted)
	auto add = [&](float2 p) {
		const float now = fmaxf(top, p.x);
		sum				= (top == now ? sum : sum * exp2_native((top - now) * LOG2_E)) + (p.x == now ? p.y : p.y * exp2_native((p.x - now) * LOG2_E));
		top				= now;
	};
	auto across = [&](int first) { // lanes of a wave that have the same row
#pragma unroll
		for (int d = first; d >= ROWS; d >>= 1) {
			add(make_float2(__shfl_xor(top, d), __shfl_xor(sum, d)));
		}
	};
	if (m < M) {
		for (int i = lane; i < count; i += LANES * AT_ONCE) {
			float2 p[AT_ONCE];
#pragma unroll
			for (int j = 0; j < AT_ONCE; ++j) {
				p[j] = i + LANES * j < count ? parts[static_cast<int64_t>(i + LANES * j) * M + m] : make_float2(none, 0.0f);
			}
#pragma unroll
			for (int j = 0; j < AT_ONCE; ++j) {
				add(p[j]);
			}
		}
	}
	across(32);
	if ((threadIdx.x & 63) < ROWS) {
		all[threadIdx.x / 64][col] = make_float2(top, sum);
	}
	__syncthreads();
	if (threadIdx.x >= 64) {
		return;
	}
	top = none, sum = 0.0f;
#pragma unroll
	for (int u = 0; u < (WAVES * ROWS + 63) / 64; ++u) { // the waves' sums
		const int from = lane + u * (64 / ROWS);
		add(from < WAVES ? all[from][col] : make_float2(none, 0.0f));
	}
	across(32);
	if (lane == 0 && m < M) {
		const float rest = logf(sum);
		lse[m]			 = top + rest;
		losses[m]		 = targets[m] >= 0 && targets[m] < N ? (top - hit[m]) + rest : 0.0f; // (not by lse: a small loss would be left in steps of its last place)
	}
}

constexpr int64_t up(int64_t n, int64_t to) {
	return (n + to - 1) / to * to;
}

// ---- backward ----

constexpr int MAXIMA = 64;
__global__ __launch_bounds__(1024) void i8_largest_scales(const float* scale, int n, float* out) {
	constexpr int THREADS = 1024;
	__shared__ float tops[THREADS / 64];
	float top = 0.0f;
#pragma unroll 4
	for (int i = blockIdx.x * THREADS + threadIdx.x; i < n; i += MAXIMA * THREADS) {
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
#pragma unroll
		for (int i = 0; i < THREADS / 64; ++i) {
			top = fmaxf(top, tops[i]);
		}
		out[blockIdx.x] = top;
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
// d of a row's target, from the loss: exp(l - lse) less one would keep of a sure row's what the rounding of lse leaves (at lse 25 and 1 - p = 1e-4, 8e-3 of it)
__device__ __forceinline__ float target_slope(float loss) {
	return expm1f(-loss);
}
// e, such that 2^e (1 - exp(-loss)) is in [2^12, 2^13); where that is below 2^-16 (the sum's rounding is up to 2^-18 of it), as for that.
// However lse is rounded, the other slopes as they are computed are at most a little over twice that.  lse is the largest logit plus log(sum), log(sum) >= 0, and so not below the largest once it is
// rounded either: a slope is at most exp(l - largest).  If the target has the largest, that is at most sum - 1 = exp(loss) - 1, or 1; if not, it is at most 1, and 1 - exp(-loss) is 1/2 or more.
__device__ __forceinline__ int slopes_exponent(float of_target) {
	const float most = fminf(fmaxf(-of_target, 0x1p-16f), 1.0f);
	int e;
	(void)frexpf(most, &e);
	return 13 - e;
}

constexpr int TERMS = 2; // of fp16 that a slope is a sum of

// P of a piece of the vocabulary: [term][strip of 16 rows][32 n][lane], lane's eight numbers n = 16 h + 4 (lane / 16) + i at 4 h + i, row lane % 16
struct i8_slopes {
	v8h* p;
	const int32_t* targets;
	const float *losses, *lse, *maxima;
	int M, N, first_n, blocks; // of 32 n in the piece

	template<int FN, int FM> __device__ __forceinline__ void operator()(const v4i (&sums)[FN][FM], int n0, int m0, const i8_matrix& w, const i8_matrix& x, v4f*) const {
		static_assert(FN % 2 == 0);
		const int lane = threadIdx.x & 63, group = lane >> 4, block = (n0 - first_n) / 32;
		const int f	   = scales_exponent(maxima);
		const bool all = n0 + 16 * FN <= N;
		v4f sw[FN];
#pragma unroll
		for (int c = 0; c < FN; ++c) {
			sw[c] = i8_scales4(w, n0 + 16 * c + 4 * group);
		}
		// all rows' before the first store: a wait for a load is also one for the stores before it.  (A row that is not scored: finite numbers times nothing.)
		int places[FM];
		float scales[FM], belows[FM], lifts[FM], owns[FM];
#pragma unroll
		for (int i = 0; i < FM; ++i) {
			const int m		  = m0 + 16 * i + (lane & 15);
			places[i]		  = m < M ? targets[m] : -1;
			const bool scored = places[i] >= 0 && places[i] < N;
			scales[i] = scored ? x.scale[m] : 0.0f, belows[i] = scored ? lse[m] : 0.0f;
			owns[i]	 = scored ? target_slope(losses[m]) : 0.0f;
			lifts[i] = scored ? ldexpf(1.0f, slopes_exponent(owns[i])) : 0.0f;
		}
#pragma unroll
		for (int i = 0; i < FM; ++i) {
			const int strip = m0 / 16 + i;
			if (strip >= x.strips) {
				continue;
			}
			const int target = places[i];
			const float sx = scales[i], below = belows[i], lift = lifts[i];
			const bool here = target >= 0 && target < N && target >= n0 && target < n0 + 16 * FN;
#pragma unroll
			for (int b = 0; b < FN / 2; ++b) {
				if (block + b >= blocks) {
					continue;
				}
				float v[8];
#pragma unroll
				for (int h = 0; h < 2; ++h) {
#pragma unroll
					for (int e = 0; e < 4; ++e) {
						const float l = static_cast<float>(sums[2 * b + h][i][e]) * sx * sw[2 * b + h][e];
						v[4 * h + e]  = exp2_native((l - below) * LOG2_E);
					}
				}
				if (here) {
#pragma unroll
					for (int j = 0; j < 8; ++j) {
						v[j] = n0 + 32 * b + 16 * (j >> 2) + 4 * group + (j & 3) == target ? owns[i] : v[j];
					}
				}
				v8h out[TERMS];
#pragma unroll
				for (int j = 0; j < 8; ++j) {
					v[j] *= ldexpf(sw[2 * b + (j >> 2)][j & 3], f) * lift;
					if (!all) {
						v[j] = n0 + 32 * b + 16 * (j >> 2) + 4 * group + (j & 3) < N ? v[j] : 0.0f;
					}
#pragma unroll
					for (int t = 0; t < TERMS; ++t) {
						out[t][j] = static_cast<_Float16>(v[j]);
						v[j] -= static_cast<float>(out[t][j]);
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

// Eight rows n (of 32, two fragments of 16 x 64 beside each other in LDS) of a column k, for the lane's place in the A operand of v_mfma_f32_16x16x32_f16: columns 16 c + lane % 16 of the
// fragments, rows 4 (lane / 16) + i of the first and of the second.  In a group of sixteen lanes lane 2 j + h names row j, columns 8 h .. 8 h + 7 of sixteen, and lane L gets column L of all eight rows.
typedef int v2i __attribute__((ext_vector_type(2)));
__device__ __forceinline__ v2i i8_columns(const v4u* first, const v4u* second, int c, int lane) {
	const int j = (lane & 15) >> 1, row = 4 * (lane >> 4) + (j & 3);
	// (the second strip's rows lie eight further, so that the 32 lanes that are served together meet no bank twice)
	const char* at = reinterpret_cast<const char*>(j < 4 ? first : second) + (c * 16 + (j < 4 ? row : row ^ 8)) * 16 + 8 * (lane & 1);
	return __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) v2i*)(const_cast<char*>(at)));
}
// ... as fp16: 128 + q as the low byte of 0x6400 + ... is the fp16 number 1024 + 128 + q
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
__device__ __forceinline__ v4h i8_halves(int raw) {
	const uint32_t u = static_cast<uint32_t>(raw) ^ 0x80808080u;
	const v2h low = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)), high = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u));
	const v2h a = low - static_cast<_Float16>(1152.0f), b = high - static_cast<_Float16>(1152.0f);
	return v4h{ a[0], a[1], b[0], b[1] };
}
__device__ __forceinline__ v8h i8_halves(v2i raw) {
	return __builtin_shufflevector(i8_halves(raw[0]), i8_halves(raw[1]), 0, 1, 2, 3, 4, 5, 6, 7);
}

struct i8_slope_product {
	const v8h* p; // as i8_slopes leaves it
	float* out; // [split][M][columns]
	int M, columns, strips, blocks, first_block; // columns: 64 w.steps; first_block: of the vocabulary, in 32 n
	int per; // blocks of a split
	bool add;
};

// A workgroup has 512 columns x 16 FM rows of sums over its split's blocks of 32 n, a wave 64 of the columns, so that each piece of w is made fp16 by one wave only.  Blocks come through a
// ring in LDS as in i8_tile_product, and w's pieces of the next block are read and converted among the products of this one.
// FM is such that the rows' tiles are of one height, eight strips at most: 144 rows of [32000 x 4096] are 2 x 80, and take 111 us (the gradient as a whole), 140 as 2 x 128; 300 of [128256 x 4096] 754 as
// 3 x 112, 795 as 3 x 128; 30 of it 198 as 32, 220 as 64.  Bound by the card's power: a loop of the same products alone, with nothing read, converted or transferred, takes 86 % of this one's time, which
// is the rate of the library's fp16 product.
template<int FM> __global__ __launch_bounds__(512, 2) void i8_slope_kernel(i8_matrix w, i8_slope_product a, int k_tiles, int m_tiles, int splits) {
	constexpr int WAVES = 8, FK = 4, STEPS = WAVES, NF = 2 * STEPS, FRAGMENTS = NF + FM * TERMS, LOADS = FRAGMENTS / WAVES, MORE = FRAGMENTS % WAVES, RING = 4;
	constexpr int FIRST = (FM * TERMS + 1) / 2 < 4 ? FM : 4 / TERMS; // strips of P that are in registers before a block begins; the others are read in it
	__shared__ v4u ring[RING][FRAGMENTS][64];
	// each XCD has a run of tiles, the tiles of a split (which have w's rows, or P's, in common) one behind the other
	const int tiles = k_tiles * m_tiles, run = (tiles * splits + 7) >> 3, place = (blockIdx.x & 7) * run + (blockIdx.x >> 3);
	if (place >= tiles * splits) {
		return;
	}
	const int split = place / tiles, tile = place % tiles;
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	const int step0 = tile % k_tiles * STEPS, strip0 = tile / k_tiles * FM;
	const int begin = split * a.per, blocks = min(a.per, a.blocks - begin);
	// this wave's fragments of a block: [two strips of w][step], then [strip of P][term]; the first MORE waves have one more
	const bool more = wave < MORE;
	const v4u* from[LOADS + 1]; // where the next block that is asked for lies
#pragma unroll
	for (int j = 0; j < LOADS + 1; ++j) {
		const int f = j < LOADS ? wave + WAVES * j : WAVES * LOADS + min(wave, MORE - 1);
		if (f < NF) {
			from[j] = w.q + (static_cast<int64_t>(2 * (a.first_block + begin) + f / STEPS) * w.steps + min(step0 + f % STEPS, w.steps - 1)) * 64;
		} else {
			const int t = (f - NF) % TERMS, strip = min(strip0 + (f - NF) / TERMS, a.strips - 1);
			from[j]		= reinterpret_cast<const v4u*>(a.p) + ((static_cast<int64_t>(t) * a.strips + strip) * a.blocks + begin) * 64;
		}
	}
	static_assert(LOADS >= 2 && STEPS == WAVES); // so that j is which strip of w, or P
	const int whole = (w.strips >> 1) - a.first_block - begin; // blocks whose second strip there is; the last one's place meets zeros in P
	auto load = [&](int s) {
		const v4u* instead = from[0];
#pragma unroll
		for (int j = 0; j < LOADS + 1; ++j) {
			if (j < LOADS || more) {
				const v4u* at = j == 1 && s >= whole ? instead : from[j];
				load_global_to_lds_b128(at, 16 * (j == 1 ? lane ^ 8 : lane), &ring[s % RING][j < LOADS ? wave + WAVES * j : WAVES * LOADS + wave][0]);
				from[j] += j < 2 ? static_cast<int64_t>(2) * w.steps * 64 : 64;
			}
		}
	};
	auto arrive_by = [&](auto loads, int behind) { // a block is in LDS, those up to `behind` blocks after it may be on their way
		constexpr int L = decltype(loads)::value;
		if (behind >= 2) {
			i8_arrive<2 * L>();
		} else if (behind == 1) {
			i8_arrive<L>();
		} else {
			i8_arrive<0>();
		}
	};
	auto arrive = [&](int behind) {
		if (MORE && more) {
			arrive_by(std::integral_constant<int, LOADS + 1>{}, behind);
		} else {
			arrive_by(std::integral_constant<int, LOADS>{}, behind);
		}
	};
	auto read_k = [&](int s, v2i(&raw)[FK]) {
#pragma unroll
		for (int c = 0; c < FK; ++c) {
			raw[c] = i8_columns(ring[s % RING][wave], ring[s % RING][STEPS + wave], c, lane);
		}
	};
	auto read_p = [&](int s, int i, v8h(&d)[TERMS]) {
#pragma unroll
		for (int t = 0; t < TERMS; ++t) {
			d[t] = __builtin_bit_cast(v8h, ring[s % RING][NF + i * TERMS + t][lane]);
		}
	};
	v4f sums[FK][FM] = {};
	auto multiply	 = [&](const v8h(&k)[FK], int i, const v8h(&d)[TERMS]) {
		__builtin_amdgcn_s_setprio(1); // before the other wave's conversions: 3.5 % faster
#pragma unroll
		for (int t = TERMS - 1; t >= 0; --t) { // the small term first
#pragma unroll
			for (int f = 0; f < FK; ++f) {
				sums[f][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[f], d[t], sums[f][i], 0, 0, 0);
			}
		}
		__builtin_amdgcn_s_setprio(0);
	};
	v2i raw[FK];
	v8h k[2][FK], d[2][FIRST][TERMS];
	auto block = [&](int s, int h) { // block s, from registers of parity h; the next one is in LDS
		v8h late[FM - FIRST + 1][TERMS];
#pragma unroll
		for (int i = FIRST; i < FM; ++i) {
			read_p(s, i, late[i - FIRST]);
		}
		read_k(s + 1, raw);
#pragma unroll
		for (int i = 0; i < FIRST; ++i) {
			multiply(k[h], i, d[h][i]);
		}
#pragma unroll
		for (int i = 0; i < FIRST; ++i) {
			read_p(s + 1, i, d[1 - h][i]);
		}
#pragma unroll
		for (int f = 0; f < FK; ++f) {
			k[1 - h][f] = i8_halves(raw[f]);
			asm volatile("" : "+v"(k[1 - h][f])); // here: the compiler would move it behind the test for the last block, in front of the products that take it
		}
#pragma unroll
		for (int i = FIRST; i < FM; ++i) {
			multiply(k[h], i, late[i - FIRST]);
		}
	};
	if (blocks > 0) {
		constexpr int ASKED = RING - 1; // once block s + 1 is there nobody reads block s - 1 any more: block s + ASKED takes its place
		for (int s = 0; s < min(blocks, ASKED); ++s) {
			load(s);
		}
		arrive(min(blocks, ASKED) - 1);
		read_k(0, raw);
#pragma unroll
		for (int i = 0; i < FIRST; ++i) {
			read_p(0, i, d[0][i]);
		}
#pragma unroll
		for (int f = 0; f < FK; ++f) {
			k[0][f] = i8_halves(raw[f]);
		}
		auto next = [&](int s) { // block s + 1 is there, and everybody is through with block s - 1
			arrive(min(blocks, s + ASKED) - 2 - s);
			if (s + ASKED < blocks) {
				load(s + ASKED);
			}
		};
		// (behind the last block something is read that lies in LDS, and not used)
		for (int s = 0; s < blocks; ++s) {
			next(s);
			block(s, 0);
			if (++s >= blocks) {
				break;
			}
			next(s);
			block(s, 1);
		}
	}
#pragma unroll
	for (int i = 0; i < FM; ++i) {
		const int m = 16 * (strip0 + i) + (lane & 15);
		if (m >= a.M) {
			continue;
		}
#pragma unroll
		for (int f = 0; f < FK; ++f) {
			const int at = 64 * (step0 + wave) + 16 * f + 4 * (lane >> 4);
			if (at < a.columns) {
				v4f* to = reinterpret_cast<v4f*>(a.out + (static_cast<int64_t>(split) * a.M + m) * a.columns + at);
				*to		= a.add ? *to + sums[f][i] : sums[f][i];
			}
		}
	}
}

// Few rows (up to 16) of up to 512 STEPS values: logits, slopes and their product with w in one pass over w, by 16 tokens (a strip) at a time.  A wave has 64 STEPS of the columns to itself: its part of a strip
// comes by direct transfers into LDS that is its own, two strips ahead, and is used there twice, for the wave's part of the logits and, after all waves' parts have been added up, for its
// columns of the sums, which stay in registers over all of the workgroup's strips.  One barrier a strip.  Bound by memory: w is read once (5 rows of 128256 x 4096, fp32: 95
// us, 175 as two products).
template<int STEPS> __global__ __launch_bounds__(512, 2) void i8_few_slopes(i8_matrix w, i8_matrix x, const int32_t* targets, const float* losses, const float* lse, const float* maxima, float* out) {
	constexpr int WAVES = 8, SCALES = 4;
	__shared__ v4u strip[WAVES][2][STEPS][64];
	__shared__ v4i parts[2][WAVES][64];
	__shared__ v4f scales[SCALES][64]; // of a strip: the first four
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = lane >> 4, m = lane & 15;
	const int step0 = wave * STEPS, mine = max(0, min(STEPS, w.steps - step0)); // this wave's steps of K
	const int M = x.rows, N = w.rows;
	const int f = scales_exponent(maxima);
	// rows of the odd sixteens of columns lie eight further, so that the lanes of a transposing read that are served together meet no bank twice
	const int turned = lane ^ ((lane & 16) >> 1);
	v4u xs[STEPS];
#pragma unroll
	for (int s = 0; s < STEPS; ++s) {
		xs[s] = s < mine ? x.q[(step0 + s) * 64 + lane] : v4u{};
	}
	const int target  = m < M ? targets[m] : -1;
	const bool scored = target >= 0 && target < N;
	const float sx = scored ? x.scale[m] : 0.0f, below = scored ? lse[m] : 0.0f;
	const float own	 = scored ? target_slope(losses[m]) : 0.0f;
	const float lift = scored ? ldexpf(1.0f, slopes_exponent(own)) : 0.0f;
	const int stride = gridDim.x, count = (w.strips - static_cast<int>(blockIdx.x) + stride - 1) / stride; // strips of this workgroup
	asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // (from here on only transfers are counted)
	auto load = [&](int b) {
		const int at = static_cast<int>(blockIdx.x) + b * stride;
#pragma unroll
		for (int s = 0; s < STEPS; ++s) {
			load_global_to_lds_b128(w.q + (static_cast<int64_t>(at) * w.steps + min(step0 + s, w.steps - 1)) * 64, 16 * turned, &strip[wave][b & 1][s][0]);
		}
		if (wave == 0) {
			load_global_to_lds_b128(w.scale + 16 * at, 16 * min(lane, 3), &scales[b % SCALES][0]);
		}
	};
	constexpr int ALL = 15 | (7 << 4) | (3 << 14); // s_waitcnt: lgkmcnt(0) alone
	auto landed = [&](bool another) { // the strip is there; the next one may be on its way
		asm volatile("" ::: "memory");
		if (!another) {
			__builtin_amdgcn_s_waitcnt(0 | (7 << 4) | (15 << 8));
		} else if (wave == 0) {
			__builtin_amdgcn_s_waitcnt(((STEPS + 1) & 15) | (7 << 4) | (15 << 8));
		} else {
			__builtin_amdgcn_s_waitcnt((STEPS & 15) | (7 << 4) | (15 << 8));
		}
		asm volatile("" ::: "memory");
	};
	v4f sums[STEPS][4] = {};
	load(0);
	if (count > 1) {
		load(1);
	}
	for (int b = 0; b < count; ++b) {
		const auto& here = strip[wave][b & 1];
		landed(b + 1 < count);
		v4i part[2] = {};
#pragma unroll
		for (int s = 0; s < STEPS; ++s) { // (x is zero past K)
			part[s & 1] = i8_mfma(here[s][turned], xs[s], part[s & 1]);
		}
		parts[b & 1][wave][lane] = part[0] + part[1];
		asm volatile("" ::: "memory");
		__builtin_amdgcn_s_waitcnt(ALL);
		__builtin_amdgcn_s_barrier();
		asm volatile("" ::: "memory");
		v4i all = parts[b & 1][0][lane];
#pragma unroll
		for (int u = 1; u < WAVES; ++u) {
			all += parts[b & 1][u][lane];
		}
		const v4f sw = scales[b % SCALES][group];
		const int n	 = 16 * (static_cast<int>(blockIdx.x) + b * stride) + 4 * group;
		v4h p[TERMS];
#pragma unroll
		for (int e = 0; e < 4; ++e) {
			const float l = static_cast<float>(all[e]) * sx * sw[e];
			float v		  = scored && n + e == target ? own : exp2_native((l - below) * LOG2_E);
			v			  = n + e < N ? v * (ldexpf(sw[e], f) * lift) : 0.0f;
#pragma unroll
			for (int t = 0; t < TERMS; ++t) {
				p[t][e] = static_cast<_Float16>(v);
				v -= static_cast<float>(p[t][e]);
			}
		}
#pragma unroll
		for (int s = 0; s < STEPS; ++s) {
			v2i raw[2];
#pragma unroll
			for (int h = 0; h < 2; ++h) { // columns 32 h .. + 15 and + 16 .. + 31 of the step, rows 4 group + i of each
				const int j = (lane & 15) >> 1, c = 2 * h + (j >> 2), row = (4 * group + (j & 3)) ^ (8 * (j >> 2));
				const char* at = reinterpret_cast<const char*>(&here[s][0]) + (c * 16 + row) * 16 + 8 * (lane & 1);
				raw[h]		   = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) v2i*)(const_cast<char*>(at)));
			}
#pragma unroll
			for (int c = 0; c < 4; ++c) {
				const v4h k = i8_halves(raw[c >> 1][c & 1]);
#pragma unroll
				for (int t = TERMS - 1; t >= 0; --t) {
					sums[s][c] = __builtin_amdgcn_mfma_f32_16x16x16f16(k, p[t], sums[s][c], 0, 0, 0);
				}
			}
		}
		if (b + 2 < count) { // what this strip lay in is this wave's own, and has been read
			asm volatile("" ::: "memory");
			__builtin_amdgcn_s_waitcnt(ALL);
			load(b + 2);
		}
	}
	if (m < M) {
#pragma unroll
		for (int s = 0; s < STEPS; ++s) {
			if (s < mine) {
#pragma unroll
				for (int c = 0; c < 4; ++c) {
					*reinterpret_cast<v4f*>(out + (static_cast<int64_t>(blockIdx.x) * M + m) * (w.steps * I8_STEP) + 64 * (step0 + s) + 16 * c + 4 * group) = sums[s][c];
				}
			}
		}
	}
}

// the splits' sums, brought back from the powers of two, times the row's grad; LANES threads to four columns
template<int TYPE, int LANES> __global__ __launch_bounds__(256) void i8_slope_results(const float* sums, const float* maxima, const int32_t* targets, const float* losses, const float* grad,
	typename i8_type<TYPE>::store* dx, int M, int N, int K, int columns, int splits) {
	__shared__ v4f others[LANES][256 / LANES];
	const int f = scales_exponent(maxima);
	const int col = threadIdx.x % (256 / LANES), part = threadIdx.x / (256 / LANES);
	const int m = blockIdx.x * gridDim.y + blockIdx.y, k = 4 * (blockIdx.z * (256 / LANES) + col);
	const bool there = m < M && k < K;
	v4f all{};
	if (there) {
#pragma unroll 8
		for (int s = part; s < splits; s += LANES) {
			all += *reinterpret_cast<const v4f*>(sums + (static_cast<int64_t>(s) * M + m) * columns + k);
		}
	}
	if constexpr (LANES > 1) {
		others[part][col] = all;
		__syncthreads();
		if (part == 0) {
#pragma unroll
			for (int i = 1; i < LANES; ++i) {
				all += others[i][col];
			}
		}
	}
	if (!there || part > 0) {
		return;
	}
	const bool scored = targets[m] >= 0 && targets[m] < N;
	const int back	= scored ? -f - slopes_exponent(target_slope(losses[m])) : 0;
	const float g	= grad ? grad[m] : 1.0f;
#pragma unroll
	for (int e = 0; e < 4; ++e) {
		if (k + e < K) {
			dx[static_cast<int64_t>(m) * K + k + e] = i8_type<TYPE>::narrow(scored ? ldexpf(all[e], back) * g : 0.0f);
		}
	}
}

// some of x's rows, from a multiple of sixteen on
i8_matrix rows_of(const i8_matrix& x, int64_t first, int64_t rows) {
	return { x.q + first / I8_ROWS * x.steps * 64, x.scale + first, static_cast<int>(rows), static_cast<int>(i8_strips(rows)), x.steps };
}

// How the backward pass is cut: 8192 rows at a time, whose sums are kept; pieces of the vocabulary, whose slopes are; splits of a piece, so that the second product has some 256 workgroups.
constexpr int64_t GRADIENT_ROWS = 8192;
struct gradient_plan {
	int64_t piece, blocks; // n, blocks of 32 n
	int64_t k_tiles, m_tiles, splits;
	int64_t slopes, sums; // bytes
	int strips; // of rows in a tile
	bool few; // one pass
};
gradient_plan plan_gradient(int64_t m, int64_t n, int64_t k) {
	gradient_plan g{};
	const int64_t strips = i8_strips(m), steps = i8_steps(k);
	g.few				 = strips == 1 && steps <= 64;
	if (g.few) { // a workgroup to a CU, or to a strip
		g.splits = std::min<int64_t>(256, i8_strips(n));
		g.sums	 = up(g.splits * m * steps * I8_STEP * 4, 256);
		return g;
	}
	const int64_t row	 = strips * 16 * 2 * TERMS;
	g.piece				 = std::min(up(n, 32), std::max<int64_t>((int64_t{ 1 } << 27) / row / 256 * 256, 1024));
	g.blocks			 = g.piece / 32;
	g.k_tiles			 = (steps + 7) / 8;
	g.m_tiles			 = (strips + 7) / 8;
	g.strips			 = static_cast<int>((strips + g.m_tiles - 1) / g.m_tiles);
	g.splits			 = std::max<int64_t>(1, std::min(g.blocks / 8, 256 / (g.k_tiles * g.m_tiles)));
	g.slopes			 = up(row * g.piece, 256);
	g.sums				 = up(g.splits * m * steps * I8_STEP * 4, 256);
	return g;
}

void gradient_sums(const i8_matrix& w, const i8_matrix& x, const i8_gradient& g, const gradient_plan& plan, v8h* slopes, float* sums, const float* maxima, hipStream_t stream) {
	if (plan.few) {
		auto launch = [&](auto kernel) {
			kernel<<<static_cast<unsigned>(plan.splits), 512, 0, stream>>>(w, x, g.targets, g.losses, g.lse, maxima, sums);
		};
		w.steps <= 16 ? launch(i8_few_slopes<2>) : w.steps <= 32 ? launch(i8_few_slopes<4>) : launch(i8_few_slopes<8>);
		return;
	}
	for (int64_t first = 0; first < w.rows; first += plan.piece) {
		const int64_t n = std::min<int64_t>(plan.piece, w.rows - first), blocks = (n + 31) / 32;
		const i8_slopes epi{ slopes, g.targets, g.losses, g.lse, maxima, x.rows, w.rows, static_cast<int>(first), static_cast<int>(blocks) };
		i8_launch_product<true>(i8_form_for(i8_strips(n), x.strips, w.steps, EPILOGUE), w, x, static_cast<int>(first), static_cast<int>(n), epi, stream);
		i8_slope_product a{};
		a.p = slopes, a.out = sums;
		a.M = x.rows, a.columns = w.steps * I8_STEP, a.strips = x.strips, a.blocks = static_cast<int>(blocks), a.first_block = static_cast<int>(first / 32);
		a.per = static_cast<int>((blocks + plan.splits - 1) / plan.splits);
		a.add = first > 0;
		const int64_t m_tiles = (x.strips + plan.strips - 1) / plan.strips;
		const unsigned grid	  = i8_grid(plan.k_tiles * plan.splits, m_tiles);
		auto multiply = [&](auto kernel) {
			kernel<<<grid, 512, 0, stream>>>(w, a, static_cast<int>(plan.k_tiles), static_cast<int>(m_tiles), static_cast<int>(plan.splits));
		};
		switch (plan.strips) {
		case 8: multiply(i8_slope_kernel<8>); break;
		case 7: multiply(i8_slope_kernel<7>); break;
		case 6: multiply(i8_slope_kernel<6>); break;
		case 5: multiply(i8_slope_kernel<5>); break;
		case 4: multiply(i8_slope_kernel<4>); break;
		case 3: multiply(i8_slope_kernel<3>); break;
		case 2: multiply(i8_slope_kernel<2>); break;
		default: multiply(i8_slope_kernel<1>); break;
		}
	}
}

// Rows of the forward pass that go together: as many as leave 64 MiB of stretches, 256 at least.
struct losses_plan {
	i8_form form;
	int64_t stretches, rows;
};
losses_plan plan_losses(int64_t m, int64_t n, int64_t k) {
	losses_plan p{};
	const int64_t shortest = (n + 31) / 32, some = std::max<int64_t>((int64_t{ 1 } << 26) / (8 * shortest) / 256 * 256, 256);
	p.rows				   = std::min(m, std::max<int64_t>(some, 8192));
	p.form				   = i8_form_for(i8_strips(n), i8_strips(p.rows), i8_steps(k), EPILOGUE);
	p.stretches			   = (n + i8_stretch(p.form) - 1) / i8_stretch(p.form);
	if (p.stretches * p.rows * 8 > (int64_t{ 1 } << 26) && some < p.rows) { // (a large vocabulary)
		p.rows		= some;
		p.form		= i8_form_for(i8_strips(n), i8_strips(p.rows), i8_steps(k), EPILOGUE);
		p.stretches = (n + i8_stretch(p.form) - 1) / i8_stretch(p.form);
	}
	return p;
}

} // namespace

int64_t i8_losses_workspace(int64_t m, int64_t n, int64_t k) {
	const losses_plan p = plan_losses(m, n, k);
	return up(p.rows * 4, 256) + up(p.stretches * p.rows * 8, 256);
}

hipError_t launch_i8_losses(const i8_matrix& w, const i8_matrix& x, const i8_losses& l, hipStream_t stream) {
	const losses_plan plan = plan_losses(x.rows, w.rows, l.k);
	char* ws			   = static_cast<char*>(l.workspace);
	float* hit			   = reinterpret_cast<float*>(ws);
	float2* parts		   = reinterpret_cast<float2*>(ws + up(plan.rows * 4, 256));
	const int stretches	   = static_cast<int>(plan.stretches);
	for (int64_t first = 0; first < x.rows; first += plan.rows) { // (the last of them may be fewer, and are cut as the others)
		const i8_matrix some	= rows_of(x, first, std::min<int64_t>(plan.rows, x.rows - first));
		const int32_t* targets	= l.targets + first;
		float *losses = l.losses + first, *lse = l.lse + first;
		i8_launch_product<true>(plan.form, w, some, 0, w.rows, i8_stretches{ parts, hit, targets, some.rows, w.rows }, stream);
		auto join = [&](auto kernel, int rows, int threads) {
			kernel<<<(some.rows + rows - 1) / rows, threads, 0, stream>>>(parts, hit, targets, losses, lse, some.rows, w.rows, stretches);
		};
		if (some.rows > 256) {
			join(i8_join_stretches<8, 1024>, 8, 1024);
		} else if (stretches > 512) { // a workgroup to a row
			join(i8_join_stretches<1, 1024>, 1, 1024);
		} else {
			join(i8_join_stretches<1, 128>, 1, 128);
		}
	}
	return hipGetLastError();
}

int64_t i8_gradient_workspace(int64_t m, int64_t n, int64_t k) {
	const gradient_plan g = plan_gradient(std::min(m, GRADIENT_ROWS), n, k);
	return MAXIMA * 4 + g.slopes + g.sums;
}

hipError_t launch_i8_gradient(const i8_matrix& w, const i8_matrix& x, const i8_gradient& all, hipStream_t stream) {
	char* ws	  = static_cast<char*>(all.workspace);
	float* maxima = reinterpret_cast<float*>(ws);
	v8h* slopes	  = reinterpret_cast<v8h*>(ws + MAXIMA * 4);
	i8_largest_scales<<<MAXIMA, 1024, 0, stream>>>(w.scale, w.rows, maxima);
	const gradient_plan most = plan_gradient(std::min<int64_t>(x.rows, GRADIENT_ROWS), w.rows, all.k);
	float* sums				 = reinterpret_cast<float*>(ws + MAXIMA * 4 + most.slopes);
	for (int64_t first = 0; first < x.rows; first += GRADIENT_ROWS) {
		const i8_matrix some = rows_of(x, first, std::min<int64_t>(GRADIENT_ROWS, x.rows - first));
		i8_gradient g		 = all;
		g.targets += first, g.losses += first, g.lse += first;
		g.grad = all.grad ? all.grad + first : nullptr;
		g.dx   = static_cast<char*>(all.dx) + first * all.k * (all.type == NH_F32 ? 4 : 2);
		// (fewer rows behind others are cut as those are, which is what there is room for)
		gradient_sums(w, some, g, most, slopes, sums, maxima, stream);
		const int columns	  = w.steps * I8_STEP;
		const unsigned beside = static_cast<unsigned>(std::min(some.rows, 64));
		const bool many		  = most.splits >= 32; // then sixteen threads to four columns
		const int at_once	  = many ? 64 : 1024;
		const dim3 grid((some.rows + beside - 1) / beside, beside, static_cast<unsigned>((g.k + at_once - 1) / at_once));
		auto results = [&](auto one, auto sixteen, auto* dx) {
			(many ? sixteen : one)<<<grid, 256, 0, stream>>>(sums, maxima, g.targets, g.losses, g.grad, dx, some.rows, w.rows, g.k, columns, static_cast<int>(most.splits));
		};
		if (g.type == NH_F32) {
			results(i8_slope_results<NH_F32, 1>, i8_slope_results<NH_F32, 16>, static_cast<float*>(g.dx));
		} else if (g.type == NH_F16) {
			results(i8_slope_results<NH_F16, 1>, i8_slope_results<NH_F16, 16>, static_cast<uint16_t*>(g.dx));
		} else {
			results(i8_slope_results<NH_BF16, 1>, i8_slope_results<NH_BF16, 16>, static_cast<uint16_t*>(g.dx));
		}
	}
	return hipGetLastError();
}

} // namespace nh
