// The products of two int8 matrices with a scale per row, w [N][K] and x [M][K], as two kernels that leave what becomes of a tile of sums to an epilogue.
//
// w is the A operand of v_mfma_i32_16x16x64_i8 and x the B operand, so a lane has four sums of neighbouring n (4 (l / 16) + i) for one m (l % 16).  An epilogue gets FN x FM
// fragments of 16 x 16 sums: epi(sums, n0, m0, part), part the number of the stretch of 16 FN values of n.
#pragma once

#include "i8_device.h"

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

// Loads outstanding (of the transfers into LDS that a wave has asked for) down to N, this wave's LDS reads done, and all waves there.
template<int N> __device__ __forceinline__ void i8_arrive() {
	asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
	__builtin_amdgcn_s_barrier();
	asm volatile("" ::: "memory");
}

// Many rows: a workgroup has 16 WN FN x 16 WM FM sums, a wave 16 FN x 16 FM of them in registers.  Steps of 64 values come by direct transfers into a ring of four LDS
// buffers, three steps ahead, and from there into one of two sets of registers, one step ahead: a wave waits once a step, for transfers that were asked for three steps ago.
template<int WN, int WM, int FN, int FM, class EPI> __global__ __launch_bounds__(64 * WN * WM, 2) void i8_tile_product(i8_matrix w, i8_matrix x, int first_n, int n_tiles, int m_tiles, EPI epi) {
	constexpr int WAVES = WN * WM, NF = WN * FN, FRAGMENTS = NF + WM * FM, LOADS = FRAGMENTS / WAVES, RING = 4;
	static_assert(FRAGMENTS % WAVES == 0);
	__shared__ v4u ring[RING][FRAGMENTS][64];
	const i8_place p = i8_place_of(n_tiles, m_tiles);
	if (!p.there) {
		return;
	}
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wave % WN, wm = wave / WN;
	const int n_strip = first_n / I8_ROWS + p.n * NF, m_strip = p.m * WM * FM;
	const v4u* from[LOADS];
#pragma unroll
	for (int j = 0; j < LOADS; ++j) { // (strips past a matrix's last one: that one again, for sums that nobody takes)
		const int f = wave * LOADS + j;
		from[j]		= f < NF ? w.q + static_cast<int64_t>(min(n_strip + f, w.strips - 1)) * w.steps * 64 : x.q + static_cast<int64_t>(min(m_strip + f - NF, x.strips - 1)) * x.steps * 64;
	}
	auto load = [&](int s) {
#pragma unroll
		for (int j = 0; j < LOADS; ++j) {
			load_global_to_lds_b128(from[j] + s * 64, 16 * lane, &ring[s % RING][wave * LOADS + j][0]);
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
	const int steps = w.steps;
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
	auto arrive = [&](int s) { // step s is in LDS; so many of the steps behind it, that have been asked for, may be on their way
		const int ahead = min(steps, s + RING - 1) - 1 - s;
		if (ahead >= 2) {
			i8_arrive<2 * LOADS>();
		} else if (ahead == 1) {
			i8_arrive<LOADS>();
		} else {
			i8_arrive<0>();
		}
	};
	v4u a[2][FN], b[2][FM];
	for (int s = 0; s < min(steps, RING - 1); ++s) {
		load(s);
	}
	arrive(0);
	if (RING - 1 < steps) {
		load(RING - 1);
	}
	read(0, a[0], b[0]);
	auto step = [&](int s, v4u(&a0)[FN], v4u(&b0)[FM], v4u(&a1)[FN], v4u(&b1)[FM]) {
		if (s + 1 < steps) {
			arrive(s + 1); // (and everybody has read step s)
			if (s + RING < steps) {
				load(s + RING);
			}
			read(s + 1, a1, b1);
		}
		multiply(a0, b0);
	};
	for (int s = 0; s < steps; s += 2) {
		step(s, a[0], b[0], a[1], b[1]);
		if (s + 1 < steps) {
			step(s + 1, a[1], b[1], a[0], b[0]);
		}
	}
	epi.template operator()<FN, FM>(sums, (n_strip + wn * FN) * I8_ROWS, (m_strip + wm * FM) * I8_ROWS, w, x);
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
		epi.template operator()<EN, 1>(all, (n_strip + at * EN % FN) * I8_ROWS, (m_strip + at * EN / FN) * I8_ROWS, w, x);
	}
}

// four scales of neighbouring rows, from row n on (a multiple of four); 0 past the strips
__device__ __forceinline__ v4f i8_scales4(const i8_matrix& w, int n) {
	return n < w.strips * I8_ROWS ? *reinterpret_cast<const v4f*>(w.scale + n) : v4f{};
}

} // namespace nh
