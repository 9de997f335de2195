// Attention of few rows per sequence over its paged keys and values, gfx950: a decode step's one row, a short prompt's or a chunk's few.
//
//   out[r] = sum_j softmax_j(scale q[r] . k_j) v_j,  j <= position of row r
//
// (mega_attention's eval_time core in the reference, infra/core_traits.hpp:743-766, whose GPU body is empty.)
//
// Memory-bound: 4 * head_dim bytes of keys and values against 4 * head_dim * group operations per row.  Every key and value of a row group is read once, by
// the one wave that owns the step of 32 keys, in direct transfers to the wave's own slot of LDS, where the next step's are on their way while this one's
// products run (straight into the operand's registers, consecutive lanes are different rows of memory: 2.6 us a step); no barrier
// between the waves.  The rows of all query heads of the kv head, token after token, are the columns of the matrix instruction
// (v_mfma_f32_16x16x32), 16 of them a row group.  As in the tile kernel the products are transposed, S^T = K Q^T and O^T = V^T P^T: a lane's scores belong to
// one row, and the operand rows of K are put so that the lane holds the scores that it has to supply as P^T: result rows 4 (l / 16) + i of the two key
// tiles of a step are keys 8 (l / 16) + 4 tile + i, so operand row m of tile t takes key 8 (m / 4) + 4 t + m % 4.
//
// Work: the row groups of all sequences, each as many steps as its sequence has and a fixed number for what a row group takes beside them, stand in a
// row, and every workgroup takes an equal stretch of it, worked out on the GPU from the lengths (by every wave for itself): all workgroups are on the
// chip at once and end together, however the lengths differ.  (Pieces of one length, a workgroup each, were 15 to 30 % slower.)  A stretch that would
// cut a small row group takes it whole or leaves it (16 sequences of 256 tokens: 8.2 -> 5.6 us).  A workgroup's four waves take the steps of a row group in
// turn and join their results in LDS.  Where a row group has been cut, each workgroup puts its result into the workspace and counts itself; the last to
// do so joins them, in the pieces' order, so the result does not hang on who that is.
//
// Measured (fp16, 32 query heads over 8 kv heads of 128): 64 sequences of up to 8192 tokens, 238 MB, 52 us; 64 of 4096, 1074 MB, 181 us: 5.9 TB/s, against 6.35 TB/s
// that a kernel which only reads reaches.  Small calls are bound by a chain of trips to memory (arguments, lengths, pages, keys) with some hundred instructions of a
// lone wave between them: one sequence of 1000 tokens (fp32 q) 8.3 us with its call, of 64 tokens 5.8, a prompt of 117 rows 6.0.
#include "attention_device.h"

#include <algorithm>

namespace nh {

namespace {

constexpr int WAVES		 = 4;
constexpr int THREADS	 = 64 * WAVES;
constexpr int STEP		 = 32; // keys of a wave's step
constexpr int COLUMNS	 = 16; // rows of a row group
constexpr int WORKGROUPS = 512; // that the chip holds at once: two per CU
// What a row group takes beside its steps (its q, its first step's way, the joins), in steps.  (Times with the launch of a graph: 64 sequences of up
// to 8192 tokens, those of up to 600 behind a shared prefix of 8192, and 64 of 1024: 6 steps 55.7, 48.3 and 42.9 us, 8: 54.0, 52.1 and 42.7, 12: 54.8, 50.2 and 44.2.)
constexpr int FIXED = 8;
// A row group of fewer steps than WHOLE is not cut (one sequence of 256 tokens: 4.7 us, in two pieces 6.1; of 512 in four 6.3, whole 6.5), others not where a piece
// would have fewer than LEAST, or than a whole stretch (64 sequences of up to 8192 tokens: 8 steps 57.1 us, 24: 58.6).
constexpr int WHOLE = 14;
constexpr int LEAST = 8;

struct rows_workspace {
	// [slot][columns][D]  a piece's sums of weighted values, and [slot][columns] their maximum (log2) and the sum of the weights; slot = (2 * unit + (1 if the
	// piece is the first of its row group)) * kv_heads + kv head
	float* o;
	float2* ml;
	float* prefix_o; // [prefix piece][sequences][q_heads][D]
	float2* prefix_ml;
	int columns;
	int prefix_pieces;
	int32_t* counters; // [unit][kv_heads]  of the unit that a cut row group begins in: how many of its pieces are done; zero before and after every call
};
struct rows_cut {
	int64_t units; // workgroups per kv head: a power of two
	int64_t columns; // rows of a row group that are kept in the workspace
};
// One workgroup per CU where that is one for each row group (a prompt of 117 rows: 1.2 us less than with two per CU, of which every second one has nothing to do),
// else two (128 sequences of 256 tokens: 25 us, with one 30).
rows_cut plan_rows(bool one_each, int64_t group, int64_t kv_heads, int64_t row_groups) {
	rows_cut c{};
	c.units = 1;
	while (2 * c.units * kv_heads <= (row_groups * kv_heads > WORKGROUPS / 2 ? WORKGROUPS : WORKGROUPS / 2)) {
		c.units *= 2;
	}
	c.columns = one_each ? std::min<int64_t>(group, COLUMNS) : COLUMNS;
	return c;
}

int64_t rounded(int64_t bytes) {
	return (bytes + 255) / 256 * 256;
}
// lays the parts out behind `base`; returns the bytes they take
int64_t lay_out(char* base, const rows_cut& c, const prefix_cut& prefix, int64_t sequences, int64_t q_heads, int64_t kv_heads, int64_t head_dim, rows_workspace* w) {
	int64_t at = 0;
	auto part  = [&](int64_t bytes) {
		char* p = base + at;
		at += rounded(bytes);
		return p;
	};
	const int64_t own = 2 * c.units * kv_heads * c.columns, shared = prefix.pieces * sequences * q_heads;
	w->ml			 = reinterpret_cast<float2*>(part(own * 8));
	w->o			 = reinterpret_cast<float*>(part(own * head_dim * 4));
	w->prefix_ml	 = reinterpret_cast<float2*>(part(shared * 8));
	w->prefix_o		 = reinterpret_cast<float*>(part(shared * head_dim * 4));
	w->columns		 = static_cast<int>(c.columns);
	w->prefix_pieces = static_cast<int>(prefix.pieces);
	return at;
}

// Sum of a value over lanes 0 .. this one, by data-parallel primitives: within rows of 16 lanes, then from row to row.
__device__ __forceinline__ int scan64(int x) {
	x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false); // row_shr:1 (lanes that have no source add 0)
	x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
	x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
	x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
	x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false); // row_bcast:15 into rows 1 and 3
	x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false); // row_bcast:31 into rows 2 and 3
	return x;
}

// What a lane knows of sequence `seq`: its rows, its keys behind the prefix.
struct sequence_size {
	int first_row, rows, pos0; // packed rows first_row .. first_row + rows - 1; position of the first
	int keys;
};
__device__ __forceinline__ sequence_size size_of(const batch_view& b, int all_rows, int prefix_keys, int held, int seq) {
	sequence_size z{ 0, 0, 0, 0 };
	if (seq < b.sequences) {
		const int end = b.starts ? b.starts[seq + 1] : seq + 1, length = max(b.lengths[seq], 0);
		z.first_row	  = b.starts ? max(b.starts[seq], 0) : seq;
		z.rows		  = max(min(end, all_rows) - z.first_row, 0);
		z.pos0		  = length - (end - z.first_row);
		z.keys		  = max(0, min(length, held) - prefix_keys);
	}
	return z;
}

// Steps of a row group of a sequence: one, without a key, if it has none.
__device__ __forceinline__ int steps_of(const sequence_size& z) {
	return max(1, (z.keys + STEP - 1) / STEP);
}
__device__ __forceinline__ int row_groups_of(const sequence_size& z, int group) {
	return (z.rows * group + COLUMNS - 1) / COLUMNS;
}

// A stretch of one row group's steps.
struct segment {
	int seq, first_row, rows, pos0; // pos0: position of the sequence's first row
	int row_group, steps; // of all of the row group
	int begin; // of the row group's steps in the row of all work
};

// Results between workgroups: device-scope stores and loads (sc1), past the caches that another XCD does not see.
__device__ __forceinline__ void put4(float* p, v4f v) {
	asm volatile("global_store_dwordx4 %0, %1, off sc1" ::"v"(p), "v"(v) : "memory");
}
__device__ __forceinline__ void put2(float2* p, float2 v) {
	asm volatile("global_store_dwordx2 %0, %1, off sc1" ::"v"(p), "v"(__builtin_bit_cast(v2u, v)) : "memory");
}
// Four results at once, {maximum, sum} and four values of each: eight loads under one wait.
__device__ __forceinline__ void get_parts(const float2* const (&ml)[4], const float* const (&o)[4], float2 (&got_ml)[4], v4f (&got_o)[4]) {
	v2u m0, m1, m2, m3;
	asm volatile("global_load_dwordx2 %0, %8, off sc1\n\t"
				 "global_load_dwordx2 %1, %9, off sc1\n\t"
				 "global_load_dwordx2 %2, %10, off sc1\n\t"
				 "global_load_dwordx2 %3, %11, off sc1\n\t"
				 "global_load_dwordx4 %4, %12, off sc1\n\t"
				 "global_load_dwordx4 %5, %13, off sc1\n\t"
				 "global_load_dwordx4 %6, %14, off sc1\n\t"
				 "global_load_dwordx4 %7, %15, off sc1\n\t"
				 "s_waitcnt vmcnt(0)"
				 : "=&v"(m0), "=&v"(m1), "=&v"(m2), "=&v"(m3), "=&v"(got_o[0]), "=&v"(got_o[1]), "=&v"(got_o[2]), "=&v"(got_o[3])
				 : "v"(ml[0]), "v"(ml[1]), "v"(ml[2]), "v"(ml[3]), "v"(o[0]), "v"(o[1]), "v"(o[2]), "v"(o[3])
				 : "memory");
	got_ml[0] = __builtin_bit_cast(float2, m0), got_ml[1] = __builtin_bit_cast(float2, m1), got_ml[2] = __builtin_bit_cast(float2, m2), got_ml[3] = __builtin_bit_cast(float2, m3);
}

// Where piece x of row r of a step's keys lies in LDS: at x ^ k_swizzle(r), so that the sixteen lanes that read the same piece of sixteen rows hit
// different banks, of which there are 256 bytes.  The rows of an operand differ in bits 0, 1, 3 and 4.  (Values: rows of 64 bytes, four side by side.)
template<int D> __device__ __forceinline__ int k_swizzle(int r) {
	return D == 128 ? (r & 3) | ((r >> 1) & 12) : ((r >> 1) & 1) | ((r >> 2) & 6);
}

// 64 lanes' 16 bytes each, twice, the second time 1024 bytes further on in memory and in LDS (the instruction's offset counts for both), from offsets behind
// an address that the wave has.  As load_global_to_lds_b128.
__device__ __forceinline__ void load_2_to_lds(const void* src, uint32_t o0, uint32_t o1, const void* lds_dst) {
	const uint32_t lds_addr = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const char*)(static_cast<const char*>(lds_dst))));
	uint32_t saved_m0;
	asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %4\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %3\n\tglobal_load_lds_dwordx4 %2, %3 offset:1024\n\ts_mov_b32 m0, %0"
				 : "=&s"(saved_m0)
				 : "v"(o0), "v"(o1), "s"(src), "s"(lds_addr)
				 : "memory");
}

// the same number, of the lane or of the wave, which the compiler takes for another one
__device__ __forceinline__ int own(int x) {
	asm volatile("" : "+v"(x));
	return x;
}
__device__ __forceinline__ int same(int x) {
	asm volatile("" : "+s"(x));
	return __builtin_amdgcn_readfirstlane(x);
}

// a running result and another one, both sums of weights and of weighted values below their own maximum
struct running {
	float m, l;
	v4f o;
	__device__ __forceinline__ void add(float m2, float l2, v4f o2) {
		const float both = fmaxf(m, m2), at = both == -__builtin_inff() ? 0.0f : both;
		const float f1 = part_factor(m - at), f2 = part_factor(m2 - at);
		l = l * f1 + l2 * f2;
		o = o * f1 + o2 * f2;
		m = both;
	}
};

} // namespace

// The kernel's arguments behind the ones that arrive in registers.
struct rows_args {
	attention_args a;
	rows_workspace w;
};
constexpr int ROWS_ARGS_AT = 5 * 8 + 4 * 4; // where they are among all of them

template<int CACHE, int TYPE, int D>
__global__ __launch_bounds__(THREADS, 2) void attention_rows_kernel(const int32_t* lengths, const int32_t* page_table, const void* q_rows, const uint16_t* k_pages, const int32_t* starts,
	uint32_t shape, int first_width, int prefix_or_rows, uint32_t heads, rows_args) {
	// What the first loads take comes first, in fourteen dwords: those arrive in registers, the rest is read from memory, as far away as the data.
	// heads: kv_heads | group << 16;  shape: sequences | log2 of the page size << 21 | log2 of the units << 25 | whether starts are checked << 30 | one row per sequence << 31
	const int first_kv_heads = heads & 0xFFFF, first_group = heads >> 16, sequences = shape & 0x1FFFFF, first_page_shift = (shape >> 21) & 15;
	const bool one_each = (shape >> 31) != 0;
	const int all_rows	= one_each ? sequences : prefix_or_rows, prefix_count = one_each ? prefix_or_rows : 0; // (only a decode step has a prefix)
	const batch_view batch{ page_table, lengths, one_each ? nullptr : starts, sequences, first_width };
	using H				 = half_type<CACHE>;
	using vec			 = typename H::vec;
	constexpr int N		 = terms<CACHE, TYPE>;
	// Terms of a weight.  Two with q of the cache's type as well: rounded once to 16 bits the weights alone made results as far off as their own rounding does (bf16
	// 2.3e-3 of the result's size instead of 1.7e-3).  The products wait for memory here: decode of 64 sequences 51.8 us with one term, 51.9 with two; 8 chunks of 32 rows 13.3, 14.0.
	constexpr int W		 = N == 1 ? 2 : N;
	constexpr int STEPS	 = D / 32; // of q.k
	constexpr int DT	 = D / 16; // tiles of O^T
	constexpr int PIECES = D / 8; // 16-byte pieces of a key
	constexpr int LOADS	 = STEP * PIECES / 64; // instructions for a step's keys, and for its values
	constexpr int SLOT	 = 2 * STEP * PIECES; // pieces of a step
	constexpr int Q_PIECES = TYPE == NH_F32 ? D / 4 : D / 8; // of a row of q
	__shared__ v4u slots[WAVES][SLOT];
	__shared__ v4u q_share[COLUMNS * Q_PIECES];
	__shared__ float2 join_ml[WAVES][COLUMNS];
	__shared__ int is_last;
	__shared__ not_finite<D> odd_of_wave[WAVES];

	const int first_lane = threadIdx.x & 63, first_wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	const int prefix_keys = prefix_count << first_page_shift, held = first_width << first_page_shift;
	const int log2_units  = (shape >> 25) & 15;

	// The row group's q, a part by each wave: piece x of row r at x ^ (r % 8).  Columns past the last row hold that one again; their results go nowhere.
	auto load_q = [&](int lane, int wave, int group, int64_t stride, int row0, int head0, int rest, float inverse, int rows) { // row i: token row0 + (rest + i) / group, head head0 + (rest + i) % group
#pragma unroll
		for (int j = 0; j < (COLUMNS * Q_PIECES / 64 + WAVES - 1) / WAVES; ++j) {
			const int part = j * WAVES + wave;
			if (part < COLUMNS * Q_PIECES / 64) {
				const int at = 64 * part + lane, r = at / Q_PIECES, x = (at % Q_PIECES) ^ (r & 7);
				const int i = rest + min(r, rows - 1), tok = static_cast<int>((static_cast<float>(i) + 0.5f) * inverse);
				const int64_t from = (row0 + tok) * stride + static_cast<int64_t>(head0 + i - tok * group) * D;
				load_global_to_lds_b128(static_cast<const char*>(q_rows) + from * (TYPE == NH_F32 ? 4 : 2) + 16 * x, &q_share[64 * part]);
			}
		}
	};
	// One sequence of one row group: whose q and pages these are is known ahead of its length, so all three are asked for together.
	const bool single = sequences == 1 && one_each && first_group <= COLUMNS;
	const int front	  = page_table[min(first_lane, max(first_width, 1) - 1)]; // of the first sequence (the host gives a table that can be read)
	int ids = front, first_id = 0; // lane i: page first_id + i of the sequence
	if (single) {
		load_q(first_lane, first_wave, first_group, 0, 0, blockIdx.x * first_group, 0, 0.0f, first_group); // (all of them rows of token 0)
	}
	sequence_size z = size_of(batch, all_rows, prefix_keys, held, first_lane);
	// Offsets of a step's pieces (see load_step), under the way of what has been asked for so far.
	uint32_t k_offset[4], v_offset;
#pragma unroll
	for (int i = 0; i < 4; ++i) {
		k_offset[i] = D == 128 ? (first_lane >> 4) * 256 + 16 * ((first_lane & 15) ^ (first_lane >> 4) ^ (4 * i)) : (first_lane >> 3) * 128 + 16 * ((first_lane & 7) ^ ((first_lane >> 4) & 1) ^ (2 * i));
		asm volatile("" : "+v"(k_offset[i]));
	}
	v_offset = 2 * ((first_lane >> 2) << first_page_shift) + 16 * ((first_lane & 3) ^ (first_lane >> 4));
	asm volatile("" : "+v"(v_offset));
	// All work, in steps: 64 sequences at a time, one for each lane.  (Their number is below 2^31: checked on the host.)
	int longest = 0; // most steps that a row group of the lane's sequences has
	int steps, work, upto; // of the lane's sequence: steps of a row group, work of all, work up to its end from the lane 0's start on
	auto add_up = [&](int group) {
		steps	= steps_of(z);
		longest = max(longest, steps);
		work	= row_groups_of(z, group) * (FIXED + steps);
		upto	= scan64(work);
		return __builtin_amdgcn_readlane(upto, 63);
	};
	int total = add_up(first_group);
	for (int base = 64; base < sequences; base += 64) {
		z = size_of(batch, all_rows, prefix_keys, held, base + first_lane);
		total += add_up(first_group);
	}
	// A workgroup's stretch: all work over all workgroups, or, where that is little, about the root of the longest row group's steps, as a piece more costs its
	// join about what a turn of the waves does (one sequence, one kv head, 16384 keys: pieces of 4 steps 31 us, of 24 16; 1000 keys: of 4 8.4, of 8 9.6).
	const auto longer_than = [&](int than) {
		return __builtin_amdgcn_ballot_w64(longest > than) != 0;
	};
	const int little	  = longer_than(1024) ? 32 : longer_than(384) ? 20 : longer_than(64) ? 8 : WAVES;
	const int first_share = max((total + (1 << log2_units) - 1) >> log2_units, little);
	if (shape >> 30 & 1) { // starts that descend could have the same rows in so many sequences that their work has no 32-bit number: nothing is done then
		bool descend = false;
		for (int seq = first_lane; seq < sequences; seq += 64) {
			descend |= starts[seq + 1] < starts[seq];
		}
		if (__builtin_amdgcn_ballot_w64(descend)) {
			wait_stores_acknowledged();
			return;
		}
	}
	int at			= blockIdx.y * first_share;
	const int end	= min(at + first_share, total);
	if (at >= end) {
		wait_stores_acknowledged(); // (nothing may still be on its way into LDS when the workgroup ends)
		return;
	}
	// where the stretch begins
	int chunk = 0, before = 0; // the lanes' sequences are chunk .. chunk + 63; work in front of them
	segment p{};
	auto find = [&](int lane, int group) {
		for (;;) {
			if (sequences > 64) {
				z = size_of(batch, all_rows, prefix_keys, held, chunk + lane);
				add_up(group);
			}
			const uint64_t over = __builtin_amdgcn_ballot_w64(before + upto > at);
			if (over) {
				const int src  = __builtin_ctzll(over);
				p.seq		   = chunk + src;
				p.first_row	   = __builtin_amdgcn_readlane(z.first_row, src);
				p.rows		   = __builtin_amdgcn_readlane(z.rows, src);
				p.pos0		   = __builtin_amdgcn_readlane(z.pos0, src);
				p.steps		   = __builtin_amdgcn_readlane(steps, src);
				const int start = before + __builtin_amdgcn_readlane(upto, src) - __builtin_amdgcn_readlane(work, src); // of the sequence
				p.row_group	   = at - start < FIXED + p.steps ? 0 : (at - start) / (FIXED + p.steps);
				p.begin		   = start + p.row_group * (FIXED + p.steps) + FIXED;
				return;
			}
			before += __builtin_amdgcn_readlane(upto, 63); // (at is below the total: there is a next chunk)
			chunk += 64;
		}
	};
	// Where a stretch's end at x cuts the row group: at whole turns of the waves.
	auto cut_at = [&](int x) {
		return p.begin + ((x - p.begin + WAVES / 2) & -WAVES);
	};
	for (bool again = false;;) {
		// Nothing of what follows is to be worked out ahead of this loop, as the compiler would: it would be kept in far more registers than there are.
		const int lane = own(first_lane), wave = same(first_wave), group = same(first_group), kv_heads = same(first_kv_heads), page_shift = same(first_page_shift), width = same(first_width);
		const int head = same(blockIdx.x), unit = same(blockIdx.y), share = same(first_share), held = width << page_shift;
		const int tid = 64 * wave + lane, col = lane & 15, quarter = lane >> 4, q_heads = group * kv_heads;
		// (the other arguments are read here and no earlier, where the compiler would wait for them in front of the lengths)
		const auto at_args = reinterpret_cast<uintptr_t>(__builtin_amdgcn_kernarg_segment_ptr()) + ROWS_ARGS_AT;
		const auto& late   = *reinterpret_cast<const __attribute__((address_space(4))) rows_args*>(static_cast<uintptr_t>(static_cast<uint32_t>(same(static_cast<int>(at_args)))) |
			static_cast<uintptr_t>(static_cast<uint32_t>(same(static_cast<int>(at_args >> 32)))) << 32);
		const auto& a = late.a;
		const auto& w = late.w;
		const uint16_t* const v_pages = a.cache.v;
		const int64_t q_stride		  = a.q_stride;
		const int cache_pages_here	  = a.cache.pages;
		const float scale			  = a.scale;
		const int prefix_pieces_here  = w.prefix_pieces, in_front_here = a.prefix_count; // pages that all sequences begin with, read like their own
		const int32_t* const pages_in_front = a.prefix_pages;
		find(lane, group);
		const int cache_pages = same(cache_pages_here), prefix_pieces = same(prefix_pieces_here), in_front = same(in_front_here);
		const int row_group_end = p.begin + p.steps, least = p.steps < WHOLE ? p.steps : min(share, LEAST); // (as many as it has: it is not cut)
		int segment_begin = p.begin, segment_end = row_group_end;
		if (at > p.begin) { // (only where the stretch begins)
			if (at - p.begin >= least) {
				if (row_group_end - at < least) { // the one in front takes it all
					at = row_group_end;
					if (at >= end) {
						wait_stores_acknowledged();
						return;
					}
					continue;
				}
				segment_begin = cut_at(at);
			}
		}
		if (end < row_group_end) {
			if (end - p.begin < least) { // the next one takes it all
				wait_stores_acknowledged();
				return;
			}
			if (row_group_end - end >= least) {
				segment_end = cut_at(end);
			}
		}
		if (again) {
			__syncthreads(); // (what the last row group left in LDS has been read)
		}
		again = true;
		// The pages of its first keys (in registers already if they are the first sequence's first), asked for ahead of everything else: the keys wait for them.
		const int32_t* table = page_table + static_cast<int64_t>(p.seq) * width;
		const int first_key	 = prefix_keys + (segment_begin - p.begin) * STEP;
		if (p.seq == 0 && in_front == 0 && prefix_keys + (segment_end - p.begin) * STEP <= 64 << page_shift) {
			ids = front, first_id = 0;
		} else {
			first_id = first_key >> page_shift;
			const int slot = min(first_id + lane, max(width, 1) - 1);
			ids			   = (slot < in_front ? pages_in_front : table)[slot];
		}
		__builtin_amdgcn_sched_barrier(0);
		// the row group's rows: first .. first + count - 1 of the sequence's rows * group
		const float inv_group = __builtin_amdgcn_rcpf(static_cast<float>(group));
		const int first = p.row_group * COLUMNS, count = min(COLUMNS, p.rows * group - first);
		const int first_token = p.row_group == 0 ? 0 : first / group, first_rest = first - first_token * group;
		// the token of the group's row i: (first + i) / group, as first_token + (first_rest + i) / group, whose numerator is below 2^17: exact in fp32, half a
		// numerator's step away from the next whole number
		auto token_of = [&](int i) {
			return first_token + static_cast<int>((static_cast<float>(first_rest + i) + 0.5f) * inv_group);
		};
		const bool there = col < count;
		const int token	 = token_of(min(col, count - 1));
		const int q_head = head * group + first + min(col, count - 1) - token * group;
		// keys: the sequence's own ones that the lane's row sees end at `seen`, those that some row of the group sees at most_seen, that all see at all_seen
		const int seen	   = min(held, p.pos0 + token + 1);
		const int all_seen = min(held, p.pos0 + first_token + 1), most_seen = min(held, p.pos0 + token_of(count - 1) + 1);
		const int end_key = min(prefix_keys + (segment_end - p.begin) * STEP, most_seen);
		// the units that the row group is cut over: the first piece is that of the unit in front of the first cut
		int first_unit = unit, pieces = 1;
		if (segment_begin > p.begin || segment_end < row_group_end) {
			first_unit = (p.begin + least - 1) / share;
			pieces	   = (row_group_end - least) / share - first_unit + 1;
		}

		const int page_size = 1 << page_shift;
		if (!single) { // (a single sequence has one row group: it has been asked for)
			load_q(lane, wave, group, q_stride, p.first_row + first_token, head * group, first_rest, inv_group, count);
		}
		// The page of the 16 keys from `key` on, -1 if there is none: of the first 64 pages from a register, of the others from memory.
		auto page_of = [&](int key) {
			if (key >= end_key) {
				return -1;
			}
			const int slot = key >> page_shift, id = slot - first_id < 64 ? __builtin_amdgcn_readlane(ids, slot - first_id) : (slot < in_front ? pages_in_front : table)[slot];
			return id >= 0 && id < cache_pages ? id : -1;
		};
		// A step's 32 keys into the wave's slot of LDS: keys, then values, 64 pieces an instruction, the pieces of a row side by side in memory so that the lanes
		// of a quad make one request of it (straight into the operand's registers consecutive lanes are different rows: that took 2.6 us for a step).
		// Instruction j holds rows (64 / PIECES) j + lane / PIECES of the keys, whose swizzle is a part of the lane's and one of j's, and columns
		// 16 j + lane / 4 of the values, whose swizzle is the lane's.
		const int64_t page_values = static_cast<int64_t>(kv_heads) * D << page_shift, head_values = static_cast<int64_t>(head) * D << page_shift;
		auto load_step			  = [&](int base, int lo, int hi) {
			 const int64_t lo_at = max(lo, 0) * page_values + head_values, hi_at = max(hi, 0) * page_values + head_values;
			 const uint16_t* const k_lo = k_pages + lo_at + (base & (page_size - 1)) * D;
			 const uint16_t* const k_hi = k_pages + hi_at + ((base + 16) & (page_size - 1)) * D;
			 v4u* const slot			= &slots[wave][0];
			 if constexpr (D == 128) {
				 load_2_to_lds(k_lo, k_offset[0], k_offset[0], slot);
				 load_2_to_lds(k_lo + 8 * D, k_offset[1], k_offset[1], slot + 2 * 64);
				 load_2_to_lds(k_hi, k_offset[2], k_offset[2], slot + 4 * 64);
				 load_2_to_lds(k_hi + 8 * D, k_offset[3], k_offset[3], slot + 6 * 64);
			 } else {
				 load_2_to_lds(k_lo, k_offset[0], k_offset[1], slot);
				 load_2_to_lds(k_hi, k_offset[2], k_offset[3], slot + 2 * 64);
			 }
			 if (page_shift > 4) { // one page
				 const uint16_t* const v_lo = v_pages + lo_at + (base & (page_size - 1));
#pragma unroll
				 for (int j = 0; j < LOADS; ++j) {
					 load_global_to_lds_b128(v_lo + ((16 * j) << page_shift), v_offset, slot + STEP * PIECES + 64 * j);
				 }
				 return;
			 }
			 const int x			 = (lane & 3) ^ (lane >> 4);
			 const uint16_t* const v = v_pages + (x & 2 ? hi_at : lo_at) + 16 * (lane >> 2) + 8 * (x & 1);
#pragma unroll
			 for (int j = 0; j < LOADS; ++j) {
				 load_global_to_lds_b128(v + 256 * j, slot + STEP * PIECES + 64 * j);
			 }
		};
		constexpr int stride = STEP * WAVES;
		int base			 = first_key + wave * STEP;
		int lo = page_of(base), hi = page_shift > 4 ? lo : page_of(base + 16);
		load_step(base, lo, hi);

		// q as the B operand: column = row, values 32 s + 8 quarter .. + 7
		vec q[N][STEPS];
		float c;
		{
			asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * LOADS) : "memory"); // this wave's part of q is there, the step behind it on its way
			__syncthreads();
			float x[STEPS][8];
			float largest = 0.0f;
			const char* mine = reinterpret_cast<const char*>(&q_share[col * Q_PIECES]);
#pragma unroll
			for (int s = 0; s < STEPS; ++s) {
				if constexpr (TYPE == NH_F32) {
#pragma unroll
					for (int h = 0; h < 2; ++h) {
						const v4f v = *reinterpret_cast<const v4f*>(mine + 16 * ((8 * s + 2 * quarter + h) ^ (col & 7)));
#pragma unroll
						for (int j = 0; j < 4; ++j) {
							x[s][4 * h + j] = v[j];
							largest			= fmaxf(largest, fabsf(v[j]));
						}
					}
				} else {
					q[0][s] = *reinterpret_cast<const vec*>(mine + 16 * ((4 * s + quarter) ^ (col & 7)));
				}
			}
			int e = 14;
			if constexpr (TYPE == NH_F32) {
				largest		   = fmaxf(largest, swap16(largest, lane));
				largest		   = fmaxf(largest, swap32(largest, lane));
				e			   = q_exponent<CACHE, TYPE>(largest);
				const float up = ldexpf(1.0f, 14 - e);
#pragma unroll
				for (int s = 0; s < STEPS; ++s) {
					if constexpr (CACHE == NH_F16) {
#pragma unroll
						for (int j = 0; j < 8; ++j) {
							x[s][j] *= up;
						}
					}
					vec t[N];
					split8<CACHE, N>(x[s], t);
#pragma unroll
					for (int n = 0; n < N; ++n) {
						q[n][s] = t[n];
					}
				}
			}
			c = ldexpf(scale * LOG2_E, e - 14);
		}

		v4f o[DT];
#pragma unroll
		for (int t = 0; t < DT; ++t) {
			o[t] = v4f{};
		}
		float m = -__builtin_inff(), l = 0.0f;
		// A step's operands: out of the slot into registers, so that the next step can be on its way into the slot under this one's arithmetic.
		vec k[2][STEPS], v[DT];
		auto read_step = [&] {
			const v4u* keys	  = &slots[wave][0];
			const v4u* values = &slots[wave][STEP * PIECES];
#pragma unroll
			for (int t = 0; t < 2; ++t) {
				const int r = 8 * (col >> 2) + 4 * t + (col & 3), swizzle = k_swizzle<D>(r);
#pragma unroll
				for (int st = 0; st < STEPS; ++st) {
					k[t][st] = __builtin_bit_cast(vec, keys[r * PIECES + ((4 * st + quarter) ^ swizzle)]);
				}
			}
#pragma unroll
			for (int dt = 0; dt < DT; ++dt) {
				const int d = 16 * dt + col;
				v[dt]		= __builtin_bit_cast(vec, values[4 * d + (quarter ^ ((d >> 2) & 3))]);
			}
		};
		auto compute = [&](int base, int lo, int hi) {
			v4f s[2];
#pragma unroll
			for (int t = 0; t < 2; ++t) {
				s[t] = v4f{};
#pragma unroll
				for (int st = 0; st < STEPS; ++st) {
#pragma unroll
					for (int n = N - 1; n >= 0; --n) { // the small terms first
						s[t] = H::mfma16(k[t][st], q[n][st], s[t]);
					}
				}
			}
			if (base + STEP > min(all_seen, end_key) || lo < 0 || hi < 0) {
				const int from	= base + 8 * quarter; // the lane's keys are from .. from + 7, of its scores and of its values
				const bool page = (quarter & 2 ? hi : lo) >= 0;
				const int n = page ? min(seen, end_key) - from : 0, n_all = page ? end_key - from : 0; // so many of them are its row's, some row's
#pragma unroll
				for (int t = 0; t < 2; ++t) {
#pragma unroll
					for (int i = 0; i < 4; ++i) {
						s[t][i] = 4 * t + i < n ? s[t][i] : -__builtin_inff();
					}
				}
				v4u keep; // no values of the others either, whatever lies there (a weight of zero times infinity is not zero)
#pragma unroll
				for (int x = 0; x < 4; ++x) {
					keep[x] = n_all >= 2 * x + 2 ? 0xFFFFFFFFu : n_all == 2 * x + 1 ? 0xFFFFu : 0u;
				}
#pragma unroll
				for (int dt = 0; dt < DT; ++dt) {
					v[dt] = __builtin_bit_cast(vec, __builtin_bit_cast(v4u, v[dt]) & keep);
				}
			}
			float top = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
			top		  = fmaxf(top, swap16(top, lane));
			top		  = fmaxf(top, swap32(top, lane)) * c;
			const float m_new = fmaxf(m, top);
			const float below = m_new == -__builtin_inff() ? 0.0f : m_new; // (no key yet: every weight is 2^-inf)
			if (__builtin_amdgcn_ballot_w64(m_new != m)) {
				const float f = exp2_fast(m - below);
				l *= f;
#pragma unroll
				for (int t = 0; t < DT; ++t) {
					o[t] *= f;
				}
				m = m_new;
			}
			const float shift = weight_bias<CACHE> - below;
			float x[8];
#pragma unroll
			for (int j = 0; j < 8; ++j) {
				x[j] = exp2_fast(fmaf(s[j >> 2][j & 3], c, shift));
				l += x[j];
			}
			vec t[W];
			split8<CACHE, W>(x, t);
#pragma unroll
			for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
				for (int n = W - 1; n >= 0; --n) {
					o[dt] = H::mfma16(v[dt], t[n], o[dt]);
				}
			}
		};

		bool strict = false; // see not_finite
		while (base < end_key) {
			const int next = base + stride, next_lo = page_of(next), next_hi = page_shift > 4 ? next_lo : page_of(next + 16);
			asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // the step is in the slot
			if (strict) {
#pragma unroll 1
				for (int j = 0; j < LOADS; ++j) {
					const int at = 64 * j + lane, d = at / 4, x = (at % 4) ^ ((d >> 2) & 3);
					odd_of_wave[wave].template take<CACHE>(reinterpret_cast<uint16_t*>(&slots[wave][STEP * PIECES + at]), d, base + 8 * x, (x & 2 ? hi : lo) < 0 ? 0 : end_key - base - 8 * x);
				}
			}
			read_step();
			asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // ... and out of it
			__builtin_amdgcn_sched_barrier(0);
			if (next < end_key) {
				load_step(next, next_lo, next_hi);
			}
			if (base >= first_key) {
				compute(base, lo, hi);
			}
			base = next, lo = next_lo, hi = next_hi;
			if (base >= end_key) {
				float nothing = 0.0f; // NaN if one of them is not finite
#pragma unroll
				for (int t = 0; t < DT; ++t) {
#pragma unroll
					for (int i = 0; i < 4; ++i) {
						nothing = fmaf(o[t][i], 0.0f, nothing);
					}
				}
				if (__builtin_expect(__builtin_amdgcn_ballot_w64(nothing != 0.0f) != 0 || strict, 0)) {
					if (!strict) { // once more, from a step in front of the first, without a key
						strict = true;
						odd_of_wave[wave].clear(lane, 64);
#pragma unroll
						for (int t = 0; t < DT; ++t) {
							o[t] = v4f{};
						}
						m = -__builtin_inff(), l = 0.0f;
						base = first_key + wave * STEP - stride, lo = -1, hi = -1;
					} else {
#pragma unroll
						for (int t = 0; t < DT; ++t) {
#pragma unroll
							for (int i = 0; i < 4; ++i) {
								o[t][i] += odd_of_wave[wave].of(16 * t + 4 * quarter + i, seen);
							}
						}
					}
				}
			}
		}
		wait_stores_acknowledged(); // (a wave without a step has one on its way all the same)

		// The pieces of the shared prefix, whose results the first piece of the row group takes in, a part by each wave.
		if (prefix_pieces > 0 && segment_begin == p.begin) {
			const int64_t row = static_cast<int64_t>(p.seq) * q_heads + q_head, rows = static_cast<int64_t>(sequences) * q_heads;
#pragma unroll 2
			for (int i = wave; i < prefix_pieces; i += WAVES) {
				const float2 ml = w.prefix_ml[i * rows + row];
				const float* from = w.prefix_o + (i * rows + row) * D + 4 * quarter;
				v4f x[DT];
#pragma unroll
				for (int dt = 0; dt < DT; ++dt) {
					x[dt] = *reinterpret_cast<const v4f*>(from + 16 * dt);
				}
				const float both = fmaxf(m, ml.x), below = both == -__builtin_inff() ? 0.0f : both;
				const float f1 = part_factor(m - below), f2 = part_factor(ml.x - below);
				m = both;
				l = l * f1 + (quarter == 0 ? ml.y * f2 : 0.0f); // (l is added up over the quarters below)
#pragma unroll
				for (int dt = 0; dt < DT; ++dt) {
					o[dt] = o[dt] * f1 + x[dt] * f2;
				}
			}
		}
		// the four waves' results into one: a thread takes four values of a row at a time
		v4f(*join_o)[DT][64] = reinterpret_cast<v4f(*)[DT][64]>(&slots[0][0]);
		static_assert(sizeof(v4f) * WAVES * DT * 64 <= sizeof(slots), "the waves' results fit where the keys were");
		l += swap16(l, lane);
		l += swap32(l, lane);
		__syncthreads(); // (every wave is through with its slots)
#pragma unroll
		for (int dt = 0; dt < DT; ++dt) {
			join_o[wave][dt][lane] = o[dt];
		}
		if (quarter == 0) {
			join_ml[wave][col] = make_float2(m, l);
		}
		__syncthreads();
		const bool alone = pieces == 1;
		// the slot of the piece in unit i
		auto slot_of = [&](int i) {
			return static_cast<int64_t>(2 * i + (i == first_unit ? 1 : 0)) * kv_heads + head;
		};
		if (there) {
			float2 ml[WAVES];
#pragma unroll
			for (int x = 0; x < WAVES; ++x) {
				ml[x] = join_ml[x][col];
			}
			const float top = fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x)), at = top == -__builtin_inff() ? 0.0f : top;
			float f[WAVES], sum = 0.0f;
#pragma unroll
			for (int x = 0; x < WAVES; ++x) {
				f[x] = part_factor(ml[x].x - at);
				sum += ml[x].y * f[x];
			}
			v4f v[DT / WAVES];
#pragma unroll
			for (int j = 0; j < DT / WAVES; ++j) {
				v4f of_wave[WAVES];
#pragma unroll
				for (int x = 0; x < WAVES; ++x) {
					of_wave[x] = join_o[x][wave + WAVES * j][lane];
				}
				v[j] = of_wave[0] * f[0] + of_wave[1] * f[1] + (of_wave[2] * f[2] + of_wave[3] * f[3]);
			}
			static_assert(WAVES == 4);
			if (alone) {
				const float inv = sum > 0.0f || sum != sum ? __builtin_amdgcn_rcpf(sum) : 0.0f; // (within 2^-23; no key at all: zeros)
				const int64_t out_at = static_cast<int64_t>((p.first_row + token) * q_heads + q_head) * D + 16 * wave + 4 * quarter; // (rows * q_heads <= 2^30)
#pragma unroll
				for (int j = 0; j < DT / WAVES; ++j) {
					store_out4<TYPE>(a.out, out_at + 16 * WAVES * j, v[j][0] * inv, v[j][1] * inv, v[j][2] * inv, v[j][3] * inv);
				}
			} else {
				const int64_t slot_row = slot_of(unit) * w.columns + col;
#pragma unroll
				for (int j = 0; j < DT / WAVES; ++j) {
					put4(w.o + slot_row * D + 16 * (wave + WAVES * j) + 4 * quarter, v[j]);
				}
				if (wave == 0 && quarter == 0) {
					put2(w.ml + slot_row, make_float2(top, sum));
				}
			}
		}
		bool join = false;
		if (!alone) {
			wait_stores_acknowledged();
			__syncthreads();
			if (tid == 0) {
				int32_t* counter = w.counters + first_unit * kv_heads + head;
				const int done	 = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
				is_last			 = done == pieces - 1;
				if (is_last) {
					__hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); // for the next call
				}
			}
			__syncthreads();
			join = is_last != 0;
		}
		if (join) {
			// Joins the row group's pieces: D / 4 threads to a row, the pieces of few rows over what threads are left.
			constexpr int LANES = D / 4, GROUPS = THREADS / LANES;
			running* parts		= reinterpret_cast<running*>(&slots[0][0]); // [GROUPS][LANES]
			static_assert(sizeof(running) * THREADS <= sizeof(slots), "the parts of the join fit where the waves' results were");
			const int part = tid % LANES, g = tid / LANES;
			const int rows_at_once = count <= 1 ? 1 : count <= 2 ? 2 : count <= 4 ? 4 : 8; // a divisor of GROUPS
			const int ways = GROUPS / rows_at_once, way = g / rows_at_once;
			for (int r0 = 0; r0 < count; r0 += rows_at_once) {
				const int r		  = r0 + g % rows_at_once;
				const bool mine	  = r < count;
				const int tok	  = token_of(min(r, count - 1));
				const int q_h	  = head * group + first + min(r, count - 1) - tok * group;
				running sum{ -__builtin_inff(), 0.0f, v4f{} };
				if (mine) {
					for (int i0 = way; i0 < pieces; i0 += 4 * ways) {
						const float2* ml[4];
						const float* o4[4];
						float2 got_ml[4];
						v4f got_o[4];
#pragma unroll
						for (int k = 0; k < 4; ++k) {
							const int64_t at = slot_of(first_unit + min(i0 + k * ways, pieces - 1)) * w.columns + r; // (past the last one: the last one again, not added)
							ml[k]			 = w.ml + at;
							o4[k]			 = w.o + at * D + 4 * part;
						}
						get_parts(ml, o4, got_ml, got_o);
#pragma unroll
						for (int k = 0; k < 4; ++k) {
							if (i0 + k * ways < pieces) {
								sum.add(got_ml[k].x, got_ml[k].y, got_o[k]);
							}
						}
					}
				}
				__syncthreads(); // (the last rows' parts have been read)
				parts[tid] = sum;
				__syncthreads();
				if (mine && way == 0) {
					for (int i = 1; i < min(ways, pieces); ++i) {
						const running& other = parts[tid + i * rows_at_once * LANES];
						sum.add(other.m, other.l, other.o);
					}
					const float inv = sum.l > 0.0f || sum.l != sum.l ? 1.0f / sum.l : 0.0f;
					store_out4<TYPE>(a.out, ((static_cast<int64_t>(p.first_row) + tok) * q_heads + q_h) * D + 4 * part, sum.o[0] * inv, sum.o[1] * inv, sum.o[2] * inv, sum.o[3] * inv);
				}
			}
		}
		at = row_group_end;
		if (at >= end) { // (also where its rest is the next unit's)
			return;
		}
	}
}

attention_needs attention_rows_needs(int64_t sequences, bool one_each, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t prefix_keys) {
	rows_workspace w;
	const rows_cut cut = plan_rows(one_each, q_heads / kv_heads, kv_heads, WORKGROUPS); // (the most that a call may have)
	return attention_needs{ lay_out(nullptr, cut, plan_prefix(sequences, q_heads / kv_heads, kv_heads, prefix_keys), sequences, q_heads, kv_heads, head_dim, &w), cut.units * kv_heads * 4 };
}
bool attention_rows_fit(int64_t rows, int64_t sequences, bool one_each, int64_t group, int64_t table_keys) {
	const int64_t row_groups = one_each ? sequences * ((group + COLUMNS - 1) / COLUMNS) : rows * group / COLUMNS + sequences;
	return row_groups * (table_keys / STEP + 1 + FIXED) < (int64_t{ 1 } << 30);
}
// the same whatever the starts are: each sequence may have all rows (double: up to 2^20 sequences, 2^26 row groups and 2^25 steps)
static bool any_starts_fit(int64_t rows, int64_t sequences, int64_t group, int64_t table_keys) {
	return static_cast<double>(sequences) * static_cast<double>(rows * group / COLUMNS + 1) * static_cast<double>(table_keys / STEP + 1 + FIXED) < 1073741824.0;
}

template<int CACHE, int TYPE, int D> static hipError_t launch_rows(const attention_args& a, hipStream_t s) {
	const int64_t group = a.q_heads / a.cache.kv_heads, sequences = a.batch.sequences;
	const bool one_each		= a.batch.starts == nullptr;
	const int64_t row_groups = one_each ? sequences * ((group + COLUMNS - 1) / COLUMNS) : a.rows * group / COLUMNS + sequences;
	const rows_cut cut		= plan_rows(one_each, group, a.cache.kv_heads, row_groups);
	const prefix_cut prefix = a.prefix_apart ? plan_prefix(sequences, group, a.cache.kv_heads, static_cast<int64_t>(a.prefix_count) << a.cache.page_shift) : prefix_cut{};
	rows_workspace w;
	(void)lay_out(static_cast<char*>(a.workspace), cut, prefix, sequences, a.q_heads, a.cache.kv_heads, D, &w);
	w.counters = a.counters;
	if (prefix.pieces > 0) {
		const hipError_t e = launch_attention_prefix(a, CACHE, TYPE, prefix, w.prefix_o, w.prefix_ml, s);
		if (e != hipSuccess) {
			return e;
		}
	}
	// (no more workgroups than the tables have keys for, four steps each at least)
	const int64_t steps		 = (static_cast<int64_t>(a.batch.width) << a.cache.page_shift) / STEP + 1 + FIXED;
	attention_args late = a;
	late.prefix_count	= one_each && !a.prefix_apart ? a.prefix_count : 0;
	const bool check_starts	= !one_each && !any_starts_fit(a.rows, sequences, group, static_cast<int64_t>(a.batch.width) << a.cache.page_shift);
	int log2_units			 = 0;
	while ((2 << log2_units) <= cut.units && (WAVES << log2_units) < row_groups * steps) {
		++log2_units;
	}
	attention_rows_kernel<CACHE, TYPE, D><<<dim3(static_cast<unsigned>(a.cache.kv_heads), 1u << log2_units), dim3(THREADS), 0, s>>>(a.batch.lengths,
		a.batch.width > 0 ? a.batch.table : a.batch.lengths, a.q, a.cache.k, a.batch.starts,
		static_cast<uint32_t>(a.batch.sequences) | static_cast<uint32_t>(a.cache.page_shift) << 21 | static_cast<uint32_t>(log2_units) << 25 | (check_starts ? 1u << 30 : 0u) | (one_each ? 1u << 31 : 0u), a.batch.width,
		one_each ? (a.prefix_apart ? a.prefix_count : 0) : a.rows, static_cast<uint32_t>(a.cache.kv_heads) | static_cast<uint32_t>(group) << 16, rows_args{ late, w });
	return hipGetLastError();
}
template<int CACHE, int TYPE> static hipError_t launch_rows(const attention_args& a, hipStream_t s) {
	return a.head_dim == 64 ? launch_rows<CACHE, TYPE, 64>(a, s) : launch_rows<CACHE, TYPE, 128>(a, s);
}

hipError_t launch_attention_rows(const attention_args& a, int cache_type, int type, hipStream_t s) {
	if (cache_type == NH_F16) {
		return type == NH_F32 ? launch_rows<NH_F16, NH_F32>(a, s) : launch_rows<NH_F16, NH_F16>(a, s);
	}
	return type == NH_F32 ? launch_rows<NH_BF16, NH_F32>(a, s) : launch_rows<NH_BF16, NH_BF16>(a, s);
}

} // namespace nh
