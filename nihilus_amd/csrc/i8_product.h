// The products of two int8 matrices with a scale per row, w [N][K] and x [M][K], as two kernels that leave what becomes of a tile of sums to an epilogue.
//
// w is the A operand of v_mfma_i32_16x16x64_i8 and x the B operand, so a lane has four sums of neighbouring n (4 (l / 16) + i) for one m (l % 16).  An epilogue gets FN x FM
// fragments of 16 x 16 sums, the first of them at n0, m0, and FN KiB of LDS that is its wave's own: epi(sums, n0, m0, w, x, scratch).
#pragma once

#include "i8_device.h"

#include <type_traits>

namespace nh {

__device__ __forceinline__ v4i i8_mfma(v4u a, v4u b, v4i c) {
	return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(v4i, a), __builtin_bit_cast(v4i, b), c, 0, 0, 0);
}

// Which tile a workgroup has.  Workgroups go to the eight XCDs in turn: each XCD gets a run of tiles, and in a run bands of eight tiles of x go through w together, so that
// the 32 workgroups which an XCD runs at a time share their operands in its L2.
struct i8_place {
	int n, m;
	bool there;
};
constexpr int I8_BAND = 8;
__device__ __forceinline__ i8_place i8_place_of(int n_tiles, int m_tiles) {
	const int all = n_tiles * m_tiles, per = (all + 7) >> 3;
	const int t = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
	if ((blockIdx.x >> 3) >= static_cast<unsigned>(per) || t >= all) {
		return { 0, 0, false };
	}
	const int band = t / (I8_BAND * n_tiles), first = band * I8_BAND, wide = min(I8_BAND, m_tiles - first), in = t - first * n_tiles;
	return { in / wide, first + in % wide, true };
}
inline unsigned i8_grid(int64_t n_tiles, int64_t m_tiles) {
	return static_cast<unsigned>((n_tiles * m_tiles + 7) / 8 * 8);
}

// Loads outstanding (of the transfers into LDS that a wave has asked for) down to N, this wave's LDS reads done, and all waves there.  The wait is the compiler's own
// instruction, not assembly: so it knows that what was read has come, and does not wait for later reads, which are under way, where that is used.
template<int N> __device__ __forceinline__ void i8_arrive() {
	asm volatile("" ::: "memory");
	__builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | ((N >> 4) << 14)); // vmcnt(N) expcnt(7: any) lgkmcnt(0)
	__builtin_amdgcn_s_barrier();
	asm volatile("" ::: "memory");
}

// Many rows: a workgroup has 16 WN FN x 16 WM FM sums, a wave 16 FN x 16 FM of them in registers.  Steps of 64 values come by direct transfers into a ring of four LDS
// buffers, three steps ahead, and from there into one of two sets of registers, one step ahead: a wave waits once a step, for transfers that were asked for three steps ago.
// KS = 2: two such groups of waves with a ring each have the two halves of K, and join their sums in LDS.
template<int WN, int WM, int FN, int FM, int KS, class EPI> __global__ __launch_bounds__(64 * WN * WM * KS, 2) void i8_tile_product(i8_matrix w, i8_matrix x, int first_n, int n_tiles, int m_tiles, EPI epi) {
	constexpr int WAVES = WN * WM, NF = WN * FN, FRAGMENTS = NF + WM * FM, LOADS = FRAGMENTS / WAVES, MORE = FRAGMENTS % WAVES, RING = 4;
	static_assert(KS == 1 || FM % 2 == 0);
	__shared__ v4u rings[KS][RING][FRAGMENTS][64];
	static_assert(WAVES * KS * FN <= KS * RING * FRAGMENTS && (KS == 1 || WAVES * FN * FM <= KS * RING * FRAGMENTS));
	const i8_place p = i8_place_of(n_tiles, m_tiles);
	if (!p.there) {
		return;
	}
	const int lane = threadIdx.x & 63, all_wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = all_wave % WAVES, part = all_wave / WAVES, wn = wave % WN, wm = wave / WN;
	const int n_strip = first_n / I8_ROWS + p.n * NF, m_strip = p.m * WM * FM;
	const int steps = (w.steps + KS - 1) / KS, first_step = part * steps, mine = min(steps, w.steps - first_step); // (the second half may be a step shorter)
	auto& ring = rings[part];
	// this wave's fragments of a step; the first MORE waves have one more
	const bool more = MORE && wave < MORE;
	const auto fragment = [&](int j) { return j < LOADS ? wave * LOADS + j : WAVES * LOADS + min(wave, MORE - 1); };
	const v4u* from[LOADS + (MORE > 0)];
#pragma unroll
	for (int j = 0; j < LOADS + (MORE > 0); ++j) { // (strips past a matrix's last one: that one again, for sums that nobody takes)
		const int f			= fragment(j);
		const int64_t strip = f < NF ? min(n_strip + f, w.strips - 1) : min(m_strip + f - NF, x.strips - 1);
		from[j]				= (f < NF ? w.q : x.q) + (strip * w.steps + min(first_step, w.steps - 1)) * 64;
	}
	auto load = [&](int s) {
		const int at = KS == 1 ? s : min(s, max(mine - 1, 0));
#pragma unroll
		for (int j = 0; j < LOADS + (MORE > 0); ++j) {
			if (j < LOADS || more) {
				load_global_to_lds_b128(from[j] + at * 64, 16 * lane, &ring[s % RING][fragment(j)][0]);
			}
		}
	};
	// all but the last so many steps' transfers done
	auto arrive_but = [&](auto steps_behind) {
		constexpr int S = decltype(steps_behind)::value;
		if (more) {
			i8_arrive<S * (LOADS + 1)>();
		} else {
			i8_arrive<S * LOADS>();
		}
	};
	auto read = [&](int s, v4u(&a)[FN], v4u(&b)[FM]) {
#pragma unroll
		for (int f = 0; f < FN; ++f) {
			a[f] = ring[s % RING][wn * FN + f][lane];
		}
#pragma unroll
		for (int f = 0; f < FM; ++f) {
			b[f] = ring[s % RING][NF + wm * FM + f][lane];
		}
	};
	v4i sums[FN][FM] = {};
	auto multiply	 = [&](const v4u(&a)[FN], const v4u(&b)[FM]) {
#pragma unroll
		for (int i = 0; i < FM; ++i) {
#pragma unroll
			for (int f = 0; f < FN; ++f) {
				sums[f][i] = i8_mfma(a[f], b[i], sums[f][i]);
			}
		}
	};
	v4u a[2][FN], b[2][FM];
	for (int s = 0; s < min(steps, RING); ++s) {
		load(s);
	}
	auto arrive = [&](int behind) { // a step is in LDS, those up to `behind` steps after it may be on their way
		if (behind >= 3) {
			arrive_but(std::integral_constant<int, 3>{});
		} else if (behind == 2) {
			arrive_but(std::integral_constant<int, 2>{});
		} else if (behind == 1) {
			arrive_but(std::integral_constant<int, 1>{});
		} else {
			i8_arrive<0>();
		}
	};
	arrive(steps - 1);
	read(0, a[0], b[0]);
	// step s is multiplied from registers while step s + 1 is read and step s + RING takes the place of s in LDS
	int s = 0;
	for (; s + 1 + RING < steps; s += 2) {
#pragma unroll
		for (int h = 0; h < 2; ++h) {
			arrive_but(std::integral_constant<int, RING - 2>{}); // step s + h + 1 is there, and everybody has read step s + h
			load(s + h + RING);
			read(s + h + 1, a[1 - h], b[1 - h]);
			multiply(a[h], b[h]);
#pragma unroll
			for (int r = 0; r < FN + FM; ++r) { // the reads among the products: in a row they would hold the wave up until LDS has taken them all
				__builtin_amdgcn_sched_group_barrier(0x008, FN * FM / (FN + FM), 0);
				__builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
			}
		}
	}
#pragma unroll 1
	for (; s < steps; s += 2) {
#pragma unroll
		for (int h = 0; h < 2; ++h) {
			if (s + h >= steps) {
				break;
			}
			if (s + h + 1 < steps) {
				arrive(min(steps, s + h + RING) - 1 - (s + h + 1));
				if (s + h + RING < steps) {
					load(s + h + RING);
				}
				read(s + h + 1, a[1 - h], b[1 - h]);
			}
			if (KS == 1 || s + h < mine) {
				multiply(a[h], b[h]);
			}
		}
	}
	__syncthreads(); // (the rings are free)
	const int n0 = (n_strip + wn * FN) * I8_ROWS, m0 = (m_strip + wm * FM) * I8_ROWS;
	v4f* scratch = reinterpret_cast<v4f*>(&rings[0][0][0][0]) + all_wave * FN * 64;
	if constexpr (KS == 1) {
		epi.template operator()<FN, FM>(sums, n0, m0, w, x, scratch);
	} else { // each group hands over the half of the columns that is the other's to finish
		v4i(*handed)[FN * FM][64] = reinterpret_cast<v4i(*)[FN * FM][64]>(&rings[0][0][0][0]);
		constexpr int H			  = FM / 2;
		v4i half[FN][H];
#pragma unroll
		for (int i = 0; i < H; ++i) {
#pragma unroll
			for (int f = 0; f < FN; ++f) {
				handed[wave][part * FN * H + i * FN + f][lane] = part ? sums[f][i] : sums[f][H + i];
			}
		}
		__syncthreads();
#pragma unroll
		for (int i = 0; i < H; ++i) {
#pragma unroll
			for (int f = 0; f < FN; ++f) {
				half[f][i] = (part ? sums[f][H + i] : sums[f][i]) + handed[wave][(1 - part) * FN * H + i * FN + f][lane];
			}
		}
		__syncthreads();
		epi.template operator()<FN, H>(half, n0, m0 + part * H * I8_ROWS, w, x, scratch);
	}
}

// Few rows: a workgroup has 16 FN x 16 FM sums, its eight waves a stretch of K each.  Fragments go from memory into registers as they are, UNROLL steps at a time; the waves' sums are joined in
// LDS and handed out again, EN x 1 fragments (neighbours along n) to a wave.
template<int FN, int FM, int UNROLL, int EN, class EPI> __global__ __launch_bounds__(512) void i8_rows_product(i8_matrix w, i8_matrix x, int first_n, int n_tiles, int m_tiles, EPI epi) {
	constexpr int WAVES = 8;
	static_assert(FN % EN == 0);
	__shared__ v4i parts[WAVES][FN * FM][64];
	const i8_place p = i8_place_of(n_tiles, m_tiles);
	if (!p.there) {
		return;
	}
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	const int n_strip = first_n / I8_ROWS + p.n * FN, m_strip = p.m * FM;
	const v4u *a[FN], *b[FM];
#pragma unroll
	for (int f = 0; f < FN; ++f) {
		a[f] = w.q + static_cast<int64_t>(min(n_strip + f, w.strips - 1)) * w.steps * 64 + lane;
	}
#pragma unroll
	for (int f = 0; f < FM; ++f) {
		b[f] = x.q + static_cast<int64_t>(min(m_strip + f, x.strips - 1)) * x.steps * 64 + lane;
	}
	const int per = (w.steps + WAVES - 1) / WAVES, end = min(w.steps, (wave + 1) * per);
	v4i sums[FN][FM] = {};
	for (int s = wave * per; s < end; s += UNROLL) {
		v4u av[UNROLL][FN], bv[UNROLL][FM];
#pragma unroll
		for (int u = 0; u < UNROLL; ++u) {
			if (s + u < end) {
#pragma unroll
				for (int f = 0; f < FN; ++f) {
					av[u][f] = a[f][(s + u) * 64];
				}
#pragma unroll
				for (int f = 0; f < FM; ++f) {
					bv[u][f] = b[f][(s + u) * 64];
				}
			}
		}
#pragma unroll
		for (int u = 0; u < UNROLL; ++u) {
			if (s + u < end) {
#pragma unroll
				for (int f = 0; f < FN; ++f) {
#pragma unroll
					for (int i = 0; i < FM; ++i) {
						sums[f][i] = i8_mfma(av[u][f], bv[u][i], sums[f][i]);
					}
				}
			}
		}
	}
#pragma unroll
	for (int f = 0; f < FN; ++f) {
#pragma unroll
		for (int i = 0; i < FM; ++i) {
			parts[wave][i * FN + f][lane] = sums[f][i];
		}
	}
	__syncthreads();
	for (int at = wave; at < FN * FM / EN; at += WAVES) {
		v4i all[EN][1];
#pragma unroll
		for (int e = 0; e < EN; ++e) {
			all[e][0] = parts[0][at * EN + e][lane];
#pragma unroll
			for (int v = 1; v < WAVES; ++v) {
				all[e][0] += parts[v][at * EN + e][lane];
			}
		}
		epi.template operator()<EN, 1>(all, (n_strip + at * EN % FN) * I8_ROWS, (m_strip + at * EN / FN) * I8_ROWS, w, x, reinterpret_cast<v4f*>(&parts[0][at * EN][0]));
	}
}

// four scales of neighbouring rows, from row n on (a multiple of four); 0 past the strips
__device__ __forceinline__ v4f i8_scales4(const i8_matrix& w, int n) {
	return n < w.strips * I8_ROWS ? *reinterpret_cast<const v4f*>(w.scale + n) : v4f{};
}

// The kernels' forms, by the tile of a workgroup (n x m).  I8_ROWS_16, _32: the kernel for few rows; _64, _128_64, _128_HALVES: tiles with K in two halves; _128_96, _128_160, _128_192: so that rows
// are not padded far (300 of [128256 x 4096]: 210 us as 3 x 128, 169 as 2 x 160) and that tiles fill rounds (640 of [8192 x 8192]: 61 / 44).
enum i8_form { I8_ROWS_16, I8_ROWS_32, I8_TILE_64, I8_TILE_128_64, I8_TILE_128_HALVES, I8_TILE_128_96, I8_TILE_128, I8_TILE_128_160, I8_TILE_128_192, I8_TILE_256 };

// The form for [n] x [m] strips of 16 and so many steps: the one with the least time by what a round of workgroups takes, `step` ns for each step, `round` ns besides, and `behind` ns for each 16 x 16
// results of a CU; a round is as many workgroups as run at once, one to a CU, or two (then, if there are no more than 256, a step takes `alone` ns).  The numbers are a fit to all forms' times at 136
// shapes of 17 to 8192 rows, 64 to 32768 n and 64 to 16384 k, results in two bytes and in four, and at 50 shapes of losses: on average the form taken is within 0.5 % of the best, at worst 8 %.
// Measured, us at [n x k], m rows, the form taken / the next best / 256 x 256 tiles:  [4096 x 4096], 64: 6.4 / 8.9 / 46; 256: 10.2 / 12 / 45; 512: 14 / 16 / 45; 1024: 20.4 / 21.7 / 45.
// [14336 x 4096], 117: 14 / 15 / 46; 512: 36 / 44 / 48; 2048: 104 (256 x 256) / 117.  [9216 x 128], 1927: 15.8 / 20.9 (256 x 256).  [5003 x 1507], 1001: 18 / 21 / 29.  [8192 x 8192], 8192: 382 (256 x 256) / 495.
inline i8_form i8_form_for(int64_t n, int64_t m, int64_t steps, int64_t behind) {
	if (m == 1) {
		return I8_ROWS_16;
	}
	struct shape {
		i8_form form;
		int64_t n, m, per_cu, step, alone, round; // per_cu: workgroups
	};
	const shape shapes[] = { { I8_ROWS_32, 2, 2, 1, 53, 53, 1100 }, { I8_TILE_64, 4, 4, 2, 174, 114, 3000 }, { I8_TILE_128_64, 8, 4, 1, 142, 142, 3350 }, { I8_TILE_128_HALVES, 8, 8, 1, 250, 250, 2520 },
		{ I8_TILE_128_96, 8, 6, 2, 450, 240, 1600 },	{ I8_TILE_128, 8, 8, 2, 500, 290, 830 },		{ I8_TILE_128_160, 8, 10, 2, 560, 270, 800 },	{ I8_TILE_128_192, 8, 12, 2, 660, 490, 630 },
		{ I8_TILE_256, 16, 16, 1, 650, 650, 2600 } };
	i8_form best = I8_TILE_256;
	int64_t least = INT64_MAX;
	for (const shape& s : shapes) {
		const int64_t tiles = (n + s.n - 1) / s.n * ((m + s.m - 1) / s.m), left = tiles % (256 * s.per_cu), results = behind * s.n * s.m;
		int64_t time		= tiles / (256 * s.per_cu) * (steps * s.step + s.round + results * s.per_cu);
		if (left) {
			time += s.round + (left <= 256 ? steps * s.alone + results : steps * s.step + results * s.per_cu);
		}
		if (time < least && (s.form == I8_TILE_256 || tiles < (int64_t{ 1 } << 21))) { // (a grid has fewer than 2^32 threads, which the largest tiles keep to at every size)
			least = time, best = s.form;
		}
	}
	return best;
}
// n that an epilogue gets at a time (16 FN), in forms whose epilogues get pairs of fragments at least
inline int i8_stretch(i8_form form) {
	return form == I8_TILE_256 ? 128 : form == I8_TILE_128 || form == I8_TILE_128_HALVES ? 64 : 32;
}

// The product of w's rows from first_n on, n of them, and x.  PAIRS: the epilogue wants fragments two by two along n.
template<bool PAIRS, class EPI> void i8_launch_product(i8_form form, const i8_matrix& w, const i8_matrix& x, int first_n, int n, const EPI& epi, hipStream_t stream) {
	const int strips = (n + 15) / 16;
	auto launch		 = [&](auto kernel, int n_strips, int m_strips, int threads) {
		const int n_tiles = (strips + n_strips - 1) / n_strips, m_tiles = (x.strips + m_strips - 1) / m_strips;
		kernel<<<i8_grid(n_tiles, m_tiles), threads, 0, stream>>>(w, x, first_n, n_tiles, m_tiles, epi);
	};
	switch (form) {
		case I8_ROWS_16:
			if constexpr (!PAIRS) {
				if (strips <= 256) { // a CU for each strip: [4096 x 4096] the same as by twos, fewer rows faster
					launch(i8_rows_product<1, 1, 8, 1, EPI>, 1, 1, 512);
					break;
				}
			}
			launch(i8_rows_product<2, 1, 8, PAIRS ? 2 : 1, EPI>, 2, 1, 512);
			break;
		case I8_ROWS_32:
			launch(i8_rows_product<2, 2, 4, PAIRS ? 2 : 1, EPI>, 2, 2, 512);
			break;
		case I8_TILE_64:
			launch(i8_tile_product<2, 2, 2, 2, 2, EPI>, 4, 4, 512);
			break;
		case I8_TILE_128_64:
			launch(i8_tile_product<4, 1, 2, 4, 2, EPI>, 8, 4, 512);
			break;
		case I8_TILE_128_HALVES:
			launch(i8_tile_product<2, 4, 4, 2, 2, EPI>, 8, 8, 1024);
			break;
		case I8_TILE_128_96:
			launch(i8_tile_product<4, 2, 2, 3, 1, EPI>, 8, 6, 512);
			break;
		case I8_TILE_128_160:
			launch(i8_tile_product<4, 2, 2, 5, 1, EPI>, 8, 10, 512);
			break;
		case I8_TILE_128_192:
			launch(i8_tile_product<4, 2, 2, 6, 1, EPI>, 8, 12, 512);
			break;
		case I8_TILE_128:
			launch(i8_tile_product<2, 4, 4, 2, 1, EPI>, 8, 8, 512);
			break;
		case I8_TILE_256:
			launch(i8_tile_product<2, 4, 8, 4, 1, EPI>, 16, 16, 512);
			break;
	}
}

} // namespace nh
