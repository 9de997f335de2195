// Attention of many rows over the same paged keys and values, gfx950: the causal attention of packed sequences' new rows, and the part of a
// decode step's attention that goes over a prefix which the whole batch shares.
//
//   out[r] = sum_j softmax_j(scale q[r] . k_j) v_j,  j <= position of row r
//
// (k.q, softmax, .v and the head merge of the reference's mega_attention core, infra/core_traits.hpp:743-766, whose GPU body is empty.)
//
// A workgroup owns 128 rows of one kv head of one sequence (of the batch, for a prefix), four waves of 32: the rows of all query heads that share the kv head,
// token after token (row = token * group + head in the group), so that keys and values are fetched once for the group and the diagonal stays short.  It walks
// the keys in tiles of 64, which direct transfers bring into one of two LDS buffers while the other one's are in use: one barrier a tile.
//
// Both products are transposed, S^T = K Q^T and O^T = V^T P^T (v_mfma_f32_32x32x16): a lane then holds scores of ONE row, the running
// maximum and sum are the lane's own (one exchange with lane ^ 32 per tile), rescaling O is a product with a number of the lane's own, and, with the rows of
// the K operand put in the right order, the lane holds exactly the scores that it has to supply as the P^T operand: no shuffle, no LDS.
// Result rows 8 (i / 4) + 4 (l / 32) + i % 4 of a lane have to be keys 16 (i / 8) + 8 (l / 32) + i % 8, so operand row m takes key m with bits
// 2 and 3 swapped.
//
// Bound by the matrix unit, and with that by power: a prompt of 8192 rows (64 query heads over 8 kv heads of 128, fp16) takes 1.13 to 1.16 ms, 0.95 to 0.97 PFLOP/s of visible pairs,
// with the matrix unit busy 54 % of the time at a clock that falls to 1.77 GHz; the library's matrix product of 8192 x 8192 x 8192 reaches 1.15.  Seven ragged prompts of up
// to 2048 rows behind up to 1500 cached keys, bf16: 117 us, 760 TFLOP/s; their diagonals and the last workgroups' ends are the rest.  The next tile's scores are
// worked out beside this one's weights, so that both units have work (8192 rows: 1.31 ms without that and without the two buffers).
//
// Where the tiles are few, the keys are split: two groups of waves in a workgroup, each half of the keys (tile buffers of their own, joined in LDS), and then pieces
// over workgroups, joined by the last one to end (512 rows behind 8192 keys, 32 / 8 heads: 125 -> 89 us).
#include "attention_device.h"

#include <algorithm>

namespace nh {

namespace {

constexpr int WAVES = 4;
constexpr int ROWS	= 32 * WAVES;
constexpr int KEYS	= 64; // of a tile

// the key (of 32) that row m of the K operand holds
__device__ __forceinline__ int key_of_row(int m) {
	return (m & 0x13) | ((m & 4) << 1) | ((m & 8) >> 1);
}
// Pieces of 16 bytes of a K tile row (head_dim values) and of a V tile row (64 keys) are permuted in LDS so that the sixteen lanes that read
// the same piece of sixteen rows at a time hit different banks, of which there are 256 bytes: rows of 256 bytes differ in bits 0 .. 3 of their number (K,
// see key_of_row, and V alike); of rows of 128 bytes two lie side by side, so bit 0 tells the halves apart and bits 1 .. 3 the rest.
template<int D> __device__ __forceinline__ int k_swizzle(int row) {
	return D == 128 ? row & 15 : (row >> 1) & 7;
}
__device__ __forceinline__ int v_swizzle(int row) {
	return (row >> 1) & 7;
}

// The weights of a row are formed below a maximum that is followed only when the scores rise above it by more than this (as a power of two): fp16
// weights stay below 2^(8 + 7), and after a row's first tiles its results are hardly ever brought below a new one.
constexpr float RISE = weight_rise;

// Results between workgroups: device scope, past the caches that another XCD does not see.
__device__ __forceinline__ void put(float* p, float x) {
	__hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float get(const float* p) {
	return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

struct tile_place {
	int seq, first_token, tokens, first_row, pos0; // the tile's rows start at first_row of tokens * group; pos0: position of the sequence's first token
	bool there;
};
// Which sequence tile `t` belongs to: every wave adds up the sequences' tiles by itself, 64 at a time.
__device__ __forceinline__ tile_place place_of_tile(const batch_view& b, int rows, int group, int t) {
	const int lane = threadIdx.x & 63;
	tile_place p{ 0, 0, 0, 0, 0, false };
	int before = 0;
	for (int base = 0; base < b.sequences; base += 64) {
		const int seq = base + lane;
		int first = 0, n = 0, end = 0;
		if (seq < b.sequences) {
			end	  = b.starts[seq + 1];
			first = max(b.starts[seq], 0);
			n	  = max(min(end, rows) - first, 0);
		}
		const int tiles = static_cast<int>((static_cast<int64_t>(n) * group + ROWS - 1) / ROWS);
		int sum			= tiles;
#pragma unroll
		for (int d = 1; d < 64; d <<= 1) {
			const int other = __shfl_up(sum, d);
			sum += lane >= d ? other : 0;
		}
		const uint64_t over = __builtin_amdgcn_ballot_w64(before + sum > t);
		if (over) {
			const int src = __builtin_ctzll(over);
			p.seq		  = base + src;
			p.first_token = __builtin_amdgcn_readlane(first, src);
			p.tokens	  = __builtin_amdgcn_readlane(n, src);
			const int k	  = t - before - (__builtin_amdgcn_readlane(sum, src) - __builtin_amdgcn_readlane(tiles, src));
			p.first_row	  = (__builtin_amdgcn_readlane(tiles, src) - 1 - k) * ROWS; // the last tiles have the most keys: first
			p.pos0		  = max(b.lengths[p.seq], 0) - (__builtin_amdgcn_readlane(end, src) - p.first_token);
			p.there		  = true;
			return p;
		}
		before += __builtin_amdgcn_readlane(sum, 63);
	}
	return p;
}

} // namespace

// Key tiles that a piece of a tile's keys has at least: 512 keys, some 8 us, against the 4 us that writing and joining the pieces take.
constexpr int PIECE_TILES = 8;

// Where the results of a tile's pieces go, as their lanes hold them: [workgroup][wave][16 DT values, maximum, sum][lane].  counters [tile]: how many of the
// pieces are done, zero before and after every call.
struct tile_pieces {
	float* parts;
	int32_t* counters;
	int pieces; // that a tile's workgroups may take
};

// Where a prefix's partial results go: piece i of the keys, row (b, query head): o [i][b][q_heads][D] unnormalised, ml the maximum and the sum.
struct prefix_out {
	float* o;
	float2* ml;
	int keys; // of a piece, a multiple of KEYS
	int row_tiles;
};

enum tile_kind { WHOLE, IN_PIECES, OVER_PREFIX }; // a workgroup has all of its rows' keys, a piece of them, a piece of the shared prefix
// PARTS: groups of four waves that have the same rows and a part of the keys each, joined in LDS at the end.
template<int CACHE, int TYPE, int D, int KIND, int PARTS>
__global__ __launch_bounds__(64 * WAVES * PARTS, (terms<CACHE, TYPE>) == 3 && PARTS == 1 ? 1 : 2) void attention_tile_kernel(attention_args a, prefix_out out, tile_pieces cut) {
	constexpr bool PREFIX = KIND == OVER_PREFIX;
	using H				= half_type<CACHE>;
	using vec			= typename H::vec;
	constexpr int N		= terms<CACHE, TYPE>;
	constexpr int STEPS = D / 16; // of q.k
	constexpr int DT	= D / 32; // tiles of O^T
	// The next tile's scores beside this one's weights; not where q alone, in two or three terms, leaves no registers for them.
	constexpr bool AHEAD = N == 1;
	constexpr int PIECES = D / 8; // 16-byte pieces of a key
	constexpr int LOADS	 = KEYS * PIECES / (64 * WAVES); // pieces of K, and of V, per thread
	struct tiles_of_part {
		v4u k[2][KEYS * PIECES]; // of tile kt in [kt % 2]
		v4u v[2][D * (KEYS / 8)];
	};
	__shared__ tiles_of_part lds[PARTS];
	__shared__ not_finite<D> odd;

	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % WAVES, part = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / WAVES;
	auto& k_tile = lds[part].k;
	auto& v_tile = lds[part].v;
	const int col = lane & 31, half = lane >> 5;
	const int group = a.q_heads / a.cache.kv_heads;
	const int head	= blockIdx.x % a.cache.kv_heads;
	const int pieces = KIND == IN_PIECES ? cut.pieces : 1;
	tile_place p{};
	int first_key = 0, piece = 0;
	if constexpr (PREFIX) {
		const int t	= blockIdx.x / a.cache.kv_heads;
		piece		= t / out.row_tiles;
		first_key	= piece * out.keys;
		p			= tile_place{ 0, 0, a.batch.sequences, t % out.row_tiles * ROWS, 0, true };
	} else {
		p = place_of_tile(a.batch, a.rows, group, blockIdx.x / a.cache.kv_heads / pieces);
		if (!p.there) {
			return;
		}
	}
	const int32_t* table = PREFIX ? a.prefix_pages : a.batch.table + static_cast<int64_t>(p.seq) * a.batch.width;
	const int width		 = PREFIX ? a.prefix_count : a.batch.width;
	const int held		 = width << a.cache.page_shift; // keys that the table has room for (below 2^31: checked on the host)
	const int all_rows	 = p.tokens * group; // (likewise)
	const int row		 = p.first_row + 32 * wave + col;
	const bool there	 = row < all_rows;
	const int token		 = row / group;
	const int q_head	 = head * group + row - token * group;
	int pos				 = -1; // of this lane's row: it sees keys 0 .. pos
	int limit, wave_min, wave_limit; // no row of the tile sees a key from limit on, none of the wave one from wave_limit on, and all of the wave's see those up to wave_min
	if constexpr (PREFIX) {
		limit = min(first_key + out.keys, held);
		pos	  = there ? min(max(a.batch.lengths[token], 0), limit) - 1 : -1;
		wave_min = there ? pos : limit, wave_limit = pos + 1;
#pragma unroll
		for (int d = 1; d < 32; d <<= 1) {
			wave_min   = min(wave_min, __shfl_xor(wave_min, d));
			wave_limit = max(wave_limit, __shfl_xor(wave_limit, d));
		}
		wave_min   = __builtin_amdgcn_readfirstlane(wave_min);
		wave_limit = __builtin_amdgcn_readfirstlane(wave_limit);
	} else {
		const int last_row	 = min(p.first_row + ROWS, all_rows) - 1;
		const int wave_first = p.first_row + 32 * wave;
		pos					 = there ? p.pos0 + token : -1;
		limit				 = max(0, min(held, p.pos0 + last_row / group + 1));
		wave_min			 = p.pos0 + wave_first / group;
		wave_limit			 = wave_first < all_rows ? p.pos0 + min(wave_first + 31, all_rows - 1) / group + 1 : 0;
	}

	int in_pieces = 1; // so many workgroups have some of the keys
	if constexpr (KIND == IN_PIECES) {
		const int all = (limit + KEYS - 1) / KEYS, of_piece = max(PIECE_TILES, (all + pieces - 1) / pieces);
		piece		  = blockIdx.x / a.cache.kv_heads % pieces;
		in_pieces	  = max(1, (all + of_piece - 1) / of_piece);
		if (piece >= in_pieces) {
			return;
		}
		first_key = piece * of_piece * KEYS;
		limit	  = min(limit, first_key + of_piece * KEYS);
	}
	// Pages: lane i holds that of the 16 keys from 16 i on of the stretch of 1024 keys that a tile is in, -1 where there is none; and the next stretch's.
	auto load_ids = [&](int stretch) {
		const int slot = (1024 * stretch + 16 * lane) >> a.cache.page_shift;
		const int id   = table[min(slot, width - 1)]; // (there are keys, so there is an entry)
		return slot < width && id >= 0 && id < a.cache.pages ? id : -1;
	};
	const int page_size		= 1 << a.cache.page_shift;
	const int64_t head_part = static_cast<int64_t>(head) * D << a.cache.page_shift;
	// What a tile's 16-byte pieces are to a thread: K rows 16 w .. 16 w + 15 are wave w's (of one page), V rows (D / 4) w on likewise.
	constexpr int K_ROWS = 64 / PIECES; // of an instruction
	uint32_t k_offset[LOADS], v_offset[LOADS]; // bytes behind the tile's first key of the wave; v: behind the wave's first row, without the part that the page size is a factor of
#pragma unroll
	for (int j = 0; j < LOADS; ++j) {
		const int r = K_ROWS * j + lane / PIECES, d = 8 * j + lane / 8; // in the wave's part
		k_offset[j] = 2 * (r * D + 8 * ((lane % PIECES) ^ k_swizzle<D>(r)));
		v_offset[j] = 2 * (d * page_size + 8 * ((lane & 7) ^ v_swizzle(d)));
	}
	auto load_k = [&](int kt, int ids) {
		const int key	  = kt * KEYS + 16 * wave;
		const int page	  = max(__builtin_amdgcn_readlane(ids, (kt & 15) * 4 + wave), 0);
		const uint16_t* at = a.cache.k + page * a.cache.page_values + head_part + static_cast<int64_t>(key & (page_size - 1)) * D;
#pragma unroll
		for (int j = 0; j < LOADS; ++j) {
			load_global_to_lds_b128(at, k_offset[j], &k_tile[kt & 1][(LOADS * wave + j) * 64]);
		}
	};
	auto load_v = [&](int kt, int ids) {
		const uint16_t* base = a.cache.v + head_part + static_cast<int64_t>(D / WAVES) * wave * page_size;
		if (page_size >= KEYS) { // the tile is in one page
			const int page	   = max(__builtin_amdgcn_readlane(ids, (kt & 15) * 4), 0);
			const uint16_t* at = base + page * a.cache.page_values + ((kt * KEYS) & (page_size - 1));
#pragma unroll
			for (int j = 0; j < LOADS; ++j) {
				load_global_to_lds_b128(at, v_offset[j], &v_tile[kt & 1][(LOADS * wave + j) * 64]);
			}
			return;
		}
#pragma unroll
		for (int j = 0; j < LOADS; ++j) {
			const int d = 8 * j + lane / 8, x = (lane & 7) ^ v_swizzle(d); // keys 8 x .. + 7 of the tile
			const int page = max(__shfl(ids, (kt & 15) * 4 + (x >> 1)), 0);
			load_global_to_lds_b128(base + page * a.cache.page_values + d * page_size + ((8 * x) & (page_size - 1)), &v_tile[kt & 1][(LOADS * wave + j) * 64]);
		}
	};

	// This part's tiles: first_tile .. end_tile - 1; all parts go round as often (the barriers are for all).
	const int all_tiles	 = max(0, (limit + KEYS - 1) / KEYS - first_key / KEYS), rounds = (all_tiles + PARTS - 1) / PARTS;
	const int first_tile = first_key / KEYS + part * rounds, end_tile = min(first_tile + rounds, first_key / KEYS + all_tiles);
	int ids = -1, next_ids = -1, stretch = 0; // that ids are of
	auto ids_of = [&](int kt) { // kt in the stretch or in the one after
		return (kt >> 4) == stretch ? ids : next_ids;
	};
	auto load_first = [&] {
		stretch = first_tile >> 4;
		if (first_tile < end_tile) {
			ids		 = load_ids(stretch);
			next_ids = load_ids(stretch + 1);
			load_k(first_tile, ids_of(first_tile));
			load_v(first_tile, ids_of(first_tile));
			if (AHEAD && first_tile + 1 < end_tile) {
				load_k(first_tile + 1, ids_of(first_tile + 1));
			}
		}
	};
	load_first();

	// q as the B operand: column = row, values 16 s + 8 half .. + 7
	vec q[N][STEPS];
	float c; // scores times c are log2 of the weights
	{
		const int64_t at = static_cast<int64_t>(p.first_token + token) * a.q_stride + static_cast<int64_t>(q_head) * D + 8 * half;
		float x[STEPS][8];
		float largest = 0.0f;
#pragma unroll
		for (int s = 0; s < STEPS; ++s) {
			load_q8<TYPE>(a.q, at + 16 * s, there, x[s]);
		}
		int e = 14;
		if constexpr (CACHE == NH_F16 && TYPE == NH_F32) {
#pragma unroll
			for (int s = 0; s < STEPS; ++s) {
#pragma unroll
				for (int j = 0; j < 8; ++j) {
					largest = fmaxf(largest, fabsf(x[s][j]));
				}
			}
			e			   = q_exponent<CACHE, TYPE>(fmaxf(largest, swap32(largest, lane)));
			const float up = ldexpf(1.0f, 14 - e);
#pragma unroll
			for (int s = 0; s < STEPS; ++s) {
#pragma unroll
				for (int j = 0; j < 8; ++j) {
					x[s][j] *= up;
				}
			}
		}
#pragma unroll
		for (int s = 0; s < STEPS; ++s) {
			vec t[N];
			split8<CACHE, N>(x[s], t);
#pragma unroll
			for (int n = 0; n < N; ++n) {
				q[n][s] = t[n];
			}
		}
		c = ldexpf(a.scale * LOG2_E, e - 14);
	}

	v16f o[DT];
	float m, l; // what the weights are below (see RISE), this lane's part of the sum of the weights
	// scores of tile kt, whose keys are in LDS
	auto scores = [&](int kt, v16f (&s)[2]) {
		const v4u* keys = k_tile[kt & 1];
		s[0] = v16f{}, s[1] = v16f{};
#pragma unroll
		for (int st = 0; st < STEPS; ++st) {
#pragma unroll
			for (int kb = 0; kb < 2; ++kb) {
				const int r = 32 * kb + key_of_row(col);
				const vec k = __builtin_bit_cast(vec, keys[r * PIECES + ((2 * st + half) ^ k_swizzle<D>(r))]);
#pragma unroll
				for (int n = N - 1; n >= 0; --n) { // the small terms first
					s[kb] = H::mfma32(k, q[n][st], s[kb]);
				}
			}
		}
	};
	bool again = false; // see not_finite
	for (;;) {
#pragma unroll
		for (int t = 0; t < DT; ++t) {
			o[t] = v16f{};
		}
		m = -__builtin_inff(), l = 0.0f;
		const int whole = again ? 0 : limit; // tiles up to here are taken as they are
		v16f s[2];
		if constexpr (AHEAD) {
			asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
		}
		__syncthreads();
		if constexpr (AHEAD) {
			scores(first_tile, s); // (without a tile: of whatever is there, for nothing)
		}
		for (int i = 0; i < rounds; ++i) {
			const int kt		   = first_tile + i;
			const bool new_stretch = (kt >> 4) != stretch;
			if (new_stretch) {
				stretch = kt >> 4;
				ids		= next_ids;
			}
			const uint32_t bad = static_cast<uint32_t>(__builtin_amdgcn_ballot_w64(ids < 0) >> ((kt & 15) * 4)) & 15u; // groups of 16 keys without a page
			// Tile kt's values and the keys asked for with them an iteration ago have come, and all waves are through with what the next ones take the place of.
			asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
			const bool mine = PARTS == 1 || kt < end_tile; // (the last round of the second part may have none)
			if (mine && (kt * KEYS + KEYS > whole || bad)) { // values of keys that no row has: nothing, whatever lies there
#pragma unroll 1
				for (int j = 0; j < LOADS; ++j) { // (each wave in what it has loaded itself)
					const int at = (LOADS * wave + j) * 64 + lane, d = at >> 3, x = (at & 7) ^ v_swizzle(d);
					const int n	 = ((bad >> (x >> 1)) & 1) ? 0 : limit - (kt * KEYS + 8 * x); // so many of the eight keys are real
					v4u v		 = v_tile[kt & 1][at];
#pragma unroll
					for (int w = 0; w < 4; ++w) {
						v[w] = n >= 2 * w + 2 ? v[w] : n == 2 * w + 1 ? v[w] & 0xFFFFu : 0u;
					}
					v_tile[kt & 1][at] = v;
					if (again) {
						odd.template take<CACHE>(reinterpret_cast<uint16_t*>(&v_tile[kt & 1][at]), d, kt * KEYS + 8 * x, 8);
					}
				}
			}
			asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
			__syncthreads();
			if (!mine) {
				continue;
			}
			if (kt + 1 + AHEAD < end_tile) {
				load_k(kt + 1 + AHEAD, ids_of(kt + 1 + AHEAD));
			}
			if (kt + 1 < end_tile) {
				load_v(kt + 1, ids_of(kt + 1));
			}
			if (new_stretch) { // (not needed before the next iteration, whose first wait it is under)
				next_ids = load_ids(stretch + 1);
			}
			if (kt * KEYS >= wave_limit) {
				continue; // (wave-uniform; the barriers are at the top)
			}
			if constexpr (!AHEAD) {
				scores(kt, s);
			}
			if (kt * KEYS + KEYS - 1 > wave_min || bad) {
#pragma unroll
				for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
					for (int i = 0; i < 16; ++i) {
						const int key = kt * KEYS + 32 * kb + 16 * (i >> 3) + 8 * half + (i & 7);
						if (key > pos || key >= limit || ((bad >> (2 * kb + (i >> 3))) & 1)) {
							s[kb][i] = -__builtin_inff();
						}
					}
				}
			}
			float top = s[0][0];
#pragma unroll
			for (int i = 1; i < 32; ++i) {
				top = fmaxf(top, s[i >> 4][i & 15]);
			}
			top = fmaxf(top, swap32(top, lane)) * c;
			if (__builtin_amdgcn_ballot_w64(top > m + RISE)) { // a larger maximum: what there is so far is brought below it
				const float m_new = fmaxf(m, top);
				const float f	  = exp2_fast(m - (m_new == -__builtin_inff() ? 0.0f : m_new));
				l *= f;
#pragma unroll
				for (int t = 0; t < DT; ++t) {
					o[t] *= f;
				}
				m = m_new;
			}
			const float shift = weight_bias<CACHE> - (m == -__builtin_inff() ? 0.0f : m); // (no key yet: every weight is 2^-inf)
			// the next tile's scores beside this one's weights: the matrix unit and the vector unit at once
			v16f next[2];
			if constexpr (AHEAD) {
				scores(kt + 1, next); // (behind the last tile: of whatever is there, for nothing)
			}
			// (q of the cache's type: weights rounded once.  Results are off by as much again as their own rounding, bf16 2.3e-3 of their size instead of 1.7e-3, fp16 2.7e-4
			// instead of 2.0e-4; two terms would double the second product: 8192 rows 1130 -> 1623 us, seven ragged prompts 117 -> 155.)
			vec t[4][N];
#pragma unroll
			for (int g = 0; g < 4; ++g) {
				float w[8];
#pragma unroll
				for (int j = 0; j < 8; ++j) {
					w[j] = exp2_fast(fmaf(s[g >> 1][8 * (g & 1) + j], c, shift));
					l += w[j];
				}
				split8<CACHE, N>(w, t[g]);
			}
			const v4u* values = v_tile[kt & 1];
#pragma unroll
			for (int g = 0; g < 4; ++g) {
#pragma unroll
				for (int dt = 0; dt < DT; ++dt) {
					const int d = 32 * dt + col;
					const vec v = __builtin_bit_cast(vec, values[d * 8 + ((2 * g + half) ^ v_swizzle(d))]);
#pragma unroll
					for (int n = N - 1; n >= 0; --n) {
						o[dt] = H::mfma32(v, t[g][n], o[dt]);
					}
				}
			}
			if constexpr (AHEAD) {
				s[0] = next[0], s[1] = next[1];
			}
		}
		float nothing = 0.0f; // NaN if one of them is not finite
#pragma unroll
		for (int t = 0; t < DT; ++t) {
#pragma unroll
			for (int i = 0; i < 16; ++i) {
				nothing = fmaf(o[t][i], 0.0f, nothing);
			}
		}
		if (again || !__syncthreads_or(nothing != 0.0f)) {
			break;
		}
		again = true;
		odd.clear(threadIdx.x, 64 * WAVES * PARTS);
		load_first();
	}
	l += swap32(l, lane);
	if constexpr (PARTS == 2) { // the second part's result into the first one's
		float* const theirs = reinterpret_cast<float*>(lds) + wave * (16 * DT + 2) * 64 + lane;
		static_assert(sizeof(float) * WAVES * (16 * DT + 2) * 64 <= sizeof(lds), "the second part's results fit where the keys were");
		__syncthreads();
		if (part == 1) {
#pragma unroll
			for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
				for (int i = 0; i < 16; ++i) {
					theirs[(16 * dt + i) * 64] = o[dt][i];
				}
			}
			theirs[16 * DT * 64]	   = m;
			theirs[(16 * DT + 1) * 64] = l;
		}
		__syncthreads();
		if (part == 1) {
			return;
		}
		const float m2 = theirs[16 * DT * 64], l2 = theirs[(16 * DT + 1) * 64];
		const float both = fmaxf(m, m2), below = both == -__builtin_inff() ? 0.0f : both;
		const float f1 = part_factor(m - below), f2 = part_factor(m2 - below);
		l = l * f1 + l2 * f2;
		m = both;
#pragma unroll
		for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
			for (int i = 0; i < 16; ++i) {
				o[dt][i] = o[dt][i] * f1 + theirs[(16 * dt + i) * 64] * f2;
			}
		}
	}
	auto odd_values_into = [&](v16f (&o)[DT]) {
		if (again) { // (the last round's barrier is behind the last note)
#pragma unroll
			for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
				for (int i = 0; i < 16; ++i) {
					o[dt][i] += odd.of(32 * dt + 8 * (i >> 2) + 4 * half + (i & 3), pos + 1);
				}
			}
		}
	};
	__shared__ int is_last;
	if (KIND == IN_PIECES && in_pieces > 1) { // (only the first part's waves are still here)
		const int tile	   = blockIdx.x / a.cache.kv_heads / pieces * a.cache.kv_heads + head;
		auto of_piece	   = [&](int i) {
			  return cut.parts + ((static_cast<int64_t>(tile) * pieces + i) * WAVES + wave) * (16 * DT + 2) * 64 + lane;
		};
		odd_values_into(o);
		float* mine = of_piece(piece);
#pragma unroll
		for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
			for (int i = 0; i < 16; ++i) {
				put(mine + (16 * dt + i) * 64, o[dt][i]);
			}
		}
		put(mine + 16 * DT * 64, m);
		put(mine + (16 * DT + 1) * 64, l);
		wait_stores_acknowledged();
		__syncthreads();
		if (threadIdx.x == 0) {
			const int done = __hip_atomic_fetch_add(cut.counters + tile, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
			is_last		   = done == in_pieces - 1;
			if (is_last) {
				__hip_atomic_store(cut.counters + tile, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); // for the next call
			}
		}
		__syncthreads();
		if (!is_last) {
			return;
		}
		// the pieces in their order, whoever joins them
		m = -__builtin_inff(), l = 0.0f;
#pragma unroll
		for (int t = 0; t < DT; ++t) {
			o[t] = v16f{};
		}
#pragma unroll 1
		for (int j = 0; j < in_pieces; ++j) {
			const float* other = of_piece(j);
			const float m2 = get(other + 16 * DT * 64), l2 = get(other + (16 * DT + 1) * 64);
			v16f o2[DT];
#pragma unroll
			for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
				for (int i = 0; i < 16; ++i) {
					o2[dt][i] = get(other + (16 * dt + i) * 64);
				}
			}
			const float both = fmaxf(m, m2), below = both == -__builtin_inff() ? 0.0f : both;
			const float f1 = part_factor(m - below), f2 = part_factor(m2 - below);
			l = l * f1 + l2 * f2;
			m = both;
#pragma unroll
			for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
				for (int i = 0; i < 16; ++i) {
					o[dt][i] = o[dt][i] * f1 + o2[dt][i] * f2;
				}
			}
		}
	} else {
		odd_values_into(o);
	}
	if (!there) {
		return;
	}
	if constexpr (PREFIX) {
		const int64_t to = (static_cast<int64_t>(piece) * a.batch.sequences + token) * a.q_heads + q_head;
		if (half == 0) {
			out.ml[to] = make_float2(m, l);
		}
#pragma unroll
		for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
			for (int i = 0; i < 16; i += 4) {
				store_out4<NH_F32>(out.o, to * D + 4 * half + 32 * dt + 2 * i, o[dt][i], o[dt][i + 1], o[dt][i + 2], o[dt][i + 3]);
			}
		}
		return;
	}
	const float inv	 = l > 0.0f || l != l ? 1.0f / l : 0.0f; // no key at all: zeros
	const int64_t at = (static_cast<int64_t>(p.first_token + token) * a.q_heads + q_head) * D + 4 * half;
#pragma unroll
	for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
		for (int i = 0; i < 16; i += 4) {
			store_out4<TYPE>(a.out, at + 32 * dt + 2 * i, o[dt][i] * inv, o[dt][i + 1] * inv, o[dt][i + 2] * inv, o[dt][i + 3] * inv);
		}
	}
}

// How a prompt's tiles are launched: `tiles` is more than there are; two parts where there is no more than a workgroup per CU, and where there are
// far fewer, pieces.
struct tiles_cut {
	int64_t tiles;
	int pieces;
	bool parts;
};
static tiles_cut plan_tiles(int64_t rows, int64_t sequences, int64_t group, int64_t kv_heads) {
	tiles_cut c{};
	c.tiles	 = rows * group / ROWS + sequences; // (each sequence adds less than a tile)
	c.parts	 = c.tiles * kv_heads <= 320; // (256 with what is counted too many)
	c.pieces = static_cast<int>(std::min<int64_t>(8, std::max<int64_t>(1, 320 / (c.tiles * kv_heads))));
	return c;
}
attention_needs attention_tiles_needs(int64_t rows, int64_t sequences, int64_t q_heads, int64_t kv_heads, int64_t head_dim) {
	const tiles_cut c = plan_tiles(rows, sequences, q_heads / kv_heads, kv_heads);
	return c.pieces > 1 ? attention_needs{ c.tiles * kv_heads * c.pieces * WAVES * (head_dim / 2 + 2) * 64 * 4, c.tiles * kv_heads * 4 } : attention_needs{ 0, 0 };
}

// (a second group of waves, or pieces, only where the workgroups are few)
bool attention_tiles_fit(int64_t rows, int64_t sequences, int64_t q_heads, int64_t kv_heads) {
	return plan_tiles(rows, sequences, q_heads / kv_heads, kv_heads).tiles * kv_heads * 64 * WAVES < GRID_THREADS;
}

template<int CACHE, int TYPE, int D, int KIND> static hipError_t launch_tiles(const attention_args& a, const prefix_out& out, const tile_pieces& cut, int64_t tiles, bool parts, hipStream_t s) {
	const dim3 grid(static_cast<unsigned>(tiles * a.cache.kv_heads * cut.pieces));
	constexpr bool FITS = D == 64 || terms<CACHE, TYPE> < 3; // (three terms of 128 values: no registers for a second wave per SIMD)
	if constexpr (FITS) {
		if (KIND != WHOLE || parts) {
			attention_tile_kernel<CACHE, TYPE, D, KIND, 2><<<grid, dim3(64 * WAVES * 2), 0, s>>>(a, out, cut);
			return hipGetLastError();
		}
	}
	if constexpr (!FITS || KIND == WHOLE) {
		attention_tile_kernel<CACHE, TYPE, D, KIND, 1><<<grid, dim3(64 * WAVES), 0, s>>>(a, out, cut);
	}
	return hipGetLastError();
}
template<int CACHE, int TYPE, int KIND> static hipError_t launch_tiles(const attention_args& a, const prefix_out& out, const tile_pieces& cut, int64_t tiles, bool parts, hipStream_t s) {
	return a.head_dim == 64 ? launch_tiles<CACHE, TYPE, 64, KIND>(a, out, cut, tiles, parts, s) : launch_tiles<CACHE, TYPE, 128, KIND>(a, out, cut, tiles, parts, s);
}
template<int KIND> static hipError_t launch_tiles(const attention_args& a, int cache_type, int type, const prefix_out& out, const tile_pieces& cut, int64_t tiles, bool parts, hipStream_t s) {
	if (cache_type == NH_F16) {
		return type == NH_F32 ? launch_tiles<NH_F16, NH_F32, KIND>(a, out, cut, tiles, parts, s) : launch_tiles<NH_F16, NH_F16, KIND>(a, out, cut, tiles, parts, s);
	}
	return type == NH_F32 ? launch_tiles<NH_BF16, NH_F32, KIND>(a, out, cut, tiles, parts, s) : launch_tiles<NH_BF16, NH_BF16, KIND>(a, out, cut, tiles, parts, s);
}

hipError_t launch_attention_tiles(const attention_args& a, int cache_type, int type, hipStream_t s) {
	const tiles_cut c		 = plan_tiles(a.rows, a.batch.sequences, a.q_heads / a.cache.kv_heads, a.cache.kv_heads);
	const int64_t key_tiles	 = (static_cast<int64_t>(a.batch.width) << a.cache.page_shift) / KEYS + 1;
	const tile_pieces pieces = { static_cast<float*>(a.workspace), a.counters, static_cast<int>(std::min<int64_t>(c.pieces, std::max<int64_t>(1, key_tiles / PIECE_TILES))) };
	if (pieces.pieces > 1 && a.workspace != nullptr) {
		return launch_tiles<IN_PIECES>(a, cache_type, type, prefix_out{}, pieces, c.tiles, true, s);
	}
	return launch_tiles<WHOLE>(a, cache_type, type, prefix_out{}, tile_pieces{ nullptr, nullptr, 1 }, c.tiles, c.parts, s);
}

prefix_cut plan_prefix(int64_t sequences, int64_t group, int64_t kv_heads, int64_t prefix_keys) {
	prefix_cut c{};
	if (prefix_keys == 0 || sequences == 0) { // (nobody to share it)
		return c;
	}
	c.row_tiles			 = (sequences * group + ROWS - 1) / ROWS;
	const int64_t wanted = std::max<int64_t>(1, 256 / (c.row_tiles * kv_heads)); // a workgroup of two parts per CU
	c.keys				 = ((prefix_keys + wanted - 1) / wanted + 2 * KEYS - 1) / (2 * KEYS) * (2 * KEYS);
	c.pieces			 = (prefix_keys + c.keys - 1) / c.keys;
	return c;
}
bool prefix_fits(const prefix_cut& cut, int64_t kv_heads) {
	return cut.pieces * cut.row_tiles * kv_heads * 64 * WAVES * 2 < GRID_THREADS;
}
hipError_t launch_attention_prefix(const attention_args& a, int cache_type, int type, const prefix_cut& cut, float* o, float2* ml, hipStream_t s) {
	return launch_tiles<OVER_PREFIX>(a, cache_type, type, prefix_out{ o, ml, static_cast<int>(cut.keys), static_cast<int>(cut.row_tiles) }, tile_pieces{ nullptr, nullptr, 1 }, cut.pieces * cut.row_tiles,
		true, s);
}

} // namespace nh
