// Attention of one row per sequence over its paged keys and values, gfx950.
//
//   out[b] = sum_j softmax_j(scale q[b] . k_j) v_j,  j < lengths[b]
//
// (mega_attention's eval_time core in the reference, infra/core_traits.hpp:743-766, whose GPU body is empty.)
//
// Memory-bound: 4 * head_dim bytes of keys and values against 4 * head_dim * group operations.  Every key and value is read once,
// straight from its page into the registers that the matrix instruction takes it from (no LDS), by the one wave that owns the key; all
// query heads of the kv head are the columns of the instruction (v_mfma_f32_16x16x32, 16 of them at a time).  As in the tile kernel the products
// are transposed, S^T = K Q^T and O^T = V^T P^T: a lane's scores belong to one head, and the operand rows of K are put so that
// the lane holds the scores that it has to supply as P^T: result rows 4 (l / 16) + i of the two key tiles of a step are keys 8 (l / 16) +
// 4 tile + i, so operand row m of tile t takes key 8 (m / 4) + 4 t + m % 4.
//
// Work: the sequences' keys are cut into pieces of the same length, worked out on the GPU from the lengths (by every workgroup for
// itself), so that about as many workgroups as the chip holds have the same work, however the lengths differ.  A piece's four waves take its
// steps of 32 keys in turn and join their results in LDS; the pieces of a sequence are joined by a second launch.  Where one piece is all that a
// sequence has, its workgroup writes the result.
// A prefix that all sequences share is left to the tile kernel, whose rows are then the heads of all sequences; its pieces are
// joined with the sequences' own.
#include "attention_device.h"

#include <algorithm>

namespace nh {

namespace {

constexpr int WAVES		 = 4;
constexpr int THREADS	 = 64 * WAVES;
constexpr int STEP		 = 32; // keys of a wave's step
constexpr int PIECE_UNIT = STEP * WAVES;
constexpr int COLUMNS	 = 16; // query heads at a time
constexpr int WORKGROUPS = 512; // that the chip holds at once: two per CU

// What the second launch needs to know of a sequence: its pieces are first .. first + count - 1
struct sequence_pieces {
	int first, count;
};
struct decode_workspace {
	sequence_pieces* pieces; // [sequences]
	float* own_o; // [piece][q_heads][D]
	float2* own_ml; // [piece][q_heads]
	float* prefix_o; // [prefix piece][sequences][q_heads][D]
	float2* prefix_ml;
};

struct own_cut {
	int64_t units; // pieces that the keys are cut into at most, beside one per sequence
	int64_t column_tiles; // of a group of query heads
};
own_cut plan_own(int64_t group, int64_t kv_heads) {
	own_cut c{};
	c.column_tiles = (group + COLUMNS - 1) / COLUMNS;
	c.units		   = std::max<int64_t>(1, WORKGROUPS / (c.column_tiles * kv_heads));
	return c;
}

int64_t rounded(int64_t bytes) {
	return (bytes + 255) / 256 * 256;
}
// lays the parts out behind `base`; returns the bytes they take
int64_t lay_out(char* base, int64_t sequences, int64_t q_heads, int64_t head_dim, int64_t own_pieces, int64_t prefix_pieces, decode_workspace* w) {
	int64_t at = 0;
	auto part  = [&](int64_t bytes) {
		char* p = base + at;
		at += rounded(bytes);
		return p;
	};
	w->pieces	 = reinterpret_cast<sequence_pieces*>(part(sequences * static_cast<int64_t>(sizeof(sequence_pieces))));
	w->own_ml	 = reinterpret_cast<float2*>(part(own_pieces * q_heads * 8));
	w->own_o	 = reinterpret_cast<float*>(part(own_pieces * q_heads * head_dim * 4));
	w->prefix_ml = reinterpret_cast<float2*>(part(prefix_pieces * sequences * q_heads * 8));
	w->prefix_o	 = reinterpret_cast<float*>(part(prefix_pieces * sequences * q_heads * head_dim * 4));
	return at;
}

// keys of its own that a sequence has
__device__ __forceinline__ int own_keys(const batch_view& b, int prefix_keys, int held, int seq) {
	return max(0, min(b.lengths[seq], held) - prefix_keys);
}

struct piece_place {
	int seq, first_key, end_key, first, count; // its keys, and its sequence's pieces
	bool there;
};
// Piece `t` of the batch: every workgroup adds the lengths up for itself, `units` pieces' worth of them making the length of a piece.
__device__ __forceinline__ piece_place place_of_piece(const batch_view& b, int prefix_keys, int held, int units, int t, int (&share)[2 * WAVES]) {
	const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
	// 1. the sum of all lengths (units of STEP keys: 32 bits hold them)
	int sum = 0;
	for (int s = tid; s < b.sequences; s += THREADS) {
		sum += (own_keys(b, prefix_keys, held, s) + STEP - 1) / STEP;
	}
#pragma unroll
	for (int d = 1; d < 64; d <<= 1) {
		sum += __shfl_xor(sum, d);
	}
	if (lane == 0) {
		share[wave] = sum;
	}
	__syncthreads();
	sum = 0;
#pragma unroll
	for (int w = 0; w < WAVES; ++w) {
		sum += share[w];
	}
	const int steps	 = max(1, ((sum + units - 1) / units + WAVES - 1) / WAVES * WAVES); // of a piece
	const int length = steps * STEP;
	// 2. the sequence that has piece t: every wave for itself, 64 sequences at a time
	piece_place p{ 0, 0, 0, 0, 0, false };
	int before = 0;
	for (int base = 0; base < b.sequences; base += 64) {
		const int seq	= base + lane;
		const int keys	= seq < b.sequences ? own_keys(b, prefix_keys, held, seq) : 0;
		const int count = (keys + length - 1) / length;
		int upto		= count;
#pragma unroll
		for (int d = 1; d < 64; d <<= 1) {
			const int other = __shfl_up(upto, d);
			upto += lane >= d ? other : 0;
		}
		const uint64_t over = __builtin_amdgcn_ballot_w64(before + upto > t);
		if (over) {
			const int src = __builtin_ctzll(over);
			p.seq		  = base + src;
			p.count		  = __builtin_amdgcn_readlane(count, src);
			p.first		  = before + __builtin_amdgcn_readlane(upto, src) - p.count;
			p.first_key	  = prefix_keys + (t - p.first) * length;
			p.end_key	  = min(p.first_key + length, prefix_keys + __builtin_amdgcn_readlane(keys, src));
			p.there		  = true;
			return p;
		}
		before += __builtin_amdgcn_readlane(upto, 63);
	}
	return p;
}

} // namespace

template<int CACHE, int TYPE, int D>
__global__ __launch_bounds__(THREADS, 2) void attention_decode_kernel(attention_args a, decode_workspace w, int units, int column_tiles) {
	using H				= half_type<CACHE>;
	using vec			= typename H::vec;
	constexpr int N		= terms<CACHE, TYPE>;
	constexpr int STEPS = D / 32; // of q.k
	constexpr int DT	= D / 16; // tiles of O^T
	__shared__ int share[2 * WAVES];
	__shared__ v4f join_o[WAVES / 2][DT][64];
	__shared__ float join_ml[WAVES / 2][2][64];

	const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
	const int col = lane & 15, quarter = lane >> 4;
	const int group		  = a.q_heads / a.cache.kv_heads;
	const int inner		  = a.cache.kv_heads * column_tiles;
	const int head		  = blockIdx.x % inner / column_tiles, ctile = blockIdx.x % column_tiles;
	const int prefix_keys = a.prefix_count << a.cache.page_shift, held = a.batch.width << a.cache.page_shift;
	const int piece		  = blockIdx.x / inner;
	const piece_place p	  = place_of_piece(a.batch, prefix_keys, held, units, piece, share);
	if (!p.there) {
		return;
	}
	const int in_group = ctile * COLUMNS + col;
	const bool there   = in_group < group;
	const int q_head   = head * group + in_group;

	// q as the B operand: column = head, values 32 s + 8 quarter .. + 7
	vec q[N][STEPS];
	float c;
	{
		const int64_t at = static_cast<int64_t>(p.seq) * a.q_stride + static_cast<int64_t>(q_head) * D + 8 * quarter;
		float x[STEPS][8];
		float largest = 0.0f;
#pragma unroll
		for (int s = 0; s < STEPS; ++s) {
			load_q8<TYPE>(a.q, at + 32 * s, there, x[s]);
#pragma unroll
			for (int j = 0; j < 8; ++j) {
				largest = fmaxf(largest, fabsf(x[s][j]));
			}
		}
		largest		= fmaxf(largest, swap16(largest));
		largest		= fmaxf(largest, swap32(largest));
		const int e = q_exponent<CACHE, TYPE>(largest);
#pragma unroll
		for (int s = 0; s < STEPS; ++s) {
			if constexpr (CACHE == NH_F16 && TYPE == NH_F32) {
#pragma unroll
				for (int j = 0; j < 8; ++j) {
					x[s][j] = ldexpf(x[s][j], 14 - e);
				}
			}
			vec t[N];
			split8<CACHE, N>(x[s], t);
#pragma unroll
			for (int n = 0; n < N; ++n) {
				q[n][s] = t[n];
			}
		}
		c = ldexpf(a.scale * LOG2_E, e - 14);
	}

	const int32_t* table = a.batch.table + static_cast<int64_t>(p.seq) * a.batch.width;
	const int page_size	 = 1 << a.cache.page_shift;
	// A step's keys base .. base + 31 lie in the pages of its two halves of 16.
	struct step_data {
		vec k[2][STEPS], v[DT];
		int base, page_lo, page_hi;
	};
	auto load_pages = [&](int base, step_data& d) {
		d.base			 = base;
		const int slot_0 = base >> a.cache.page_shift, slot_1 = (base + 16) >> a.cache.page_shift;
		d.page_lo		 = base < p.end_key ? table[slot_0] : -1;
		d.page_hi		 = base + 16 < p.end_key ? table[slot_1] : -1;
	};
	auto page_there = [&](int id) {
		return id >= 0 && id < a.cache.pages;
	};
	auto load_step = [&](step_data& d) {
		const int lo = page_there(d.page_lo) ? d.page_lo : 0, hi = page_there(d.page_hi) ? d.page_hi : 0;
		const int64_t k_page = (col & 8 ? hi : lo) * a.cache.page_values, v_page = (quarter & 2 ? hi : lo) * a.cache.page_values;
#pragma unroll
		for (int t = 0; t < 2; ++t) {
			const int key	   = (d.base + 8 * (col >> 2) + 4 * t + (col & 3)) & (page_size - 1);
			const uint16_t* at = a.cache.k + k_page + (static_cast<int64_t>(head) * page_size + key) * D + 8 * quarter;
#pragma unroll
			for (int s = 0; s < STEPS; ++s) {
				d.k[t][s] = *reinterpret_cast<const vec*>(at + 32 * s);
			}
		}
		const uint16_t* at = a.cache.v + v_page + (static_cast<int64_t>(head) * D + col) * page_size + ((d.base + 8 * quarter) & (page_size - 1));
#pragma unroll
		for (int dt = 0; dt < DT; ++dt) {
			d.v[dt] = *reinterpret_cast<const vec*>(at + static_cast<int64_t>(dt) * 16 * page_size);
		}
	};

	v4f o[DT];
#pragma unroll
	for (int t = 0; t < DT; ++t) {
		o[t] = v4f{};
	}
	float m = -__builtin_inff(), l = 0.0f;
	auto compute = [&](step_data& d) {
		v4f s[2];
#pragma unroll
		for (int t = 0; t < 2; ++t) {
			s[t] = v4f{};
#pragma unroll
			for (int st = 0; st < STEPS; ++st) {
#pragma unroll
				for (int n = N - 1; n >= 0; --n) { // the small terms first
					s[t] = H::mfma16(d.k[t][st], q[n][st], s[t]);
				}
			}
		}
		const bool lo = page_there(d.page_lo), hi = page_there(d.page_hi);
		if (d.base + STEP > p.end_key || !lo || !hi) {
			const int first = d.base + 8 * quarter; // the lane's keys are first .. first + 7, of its scores and of its values
			const int n		= (quarter & 2 ? hi : lo) ? p.end_key - first : 0; // so many of them are real
#pragma unroll
			for (int t = 0; t < 2; ++t) {
#pragma unroll
				for (int i = 0; i < 4; ++i) {
					s[t][i] = 4 * t + i < n ? s[t][i] : -__builtin_inff();
				}
			}
#pragma unroll
			for (int dt = 0; dt < DT; ++dt) { // no values of the others either, whatever lies there (a weight of zero times infinity is not zero)
				v4u v = __builtin_bit_cast(v4u, d.v[dt]);
#pragma unroll
				for (int x = 0; x < 4; ++x) {
					v[x] = n >= 2 * x + 2 ? v[x] : n == 2 * x + 1 ? v[x] & 0xFFFFu : 0u;
				}
				d.v[dt] = __builtin_bit_cast(vec, v);
			}
		}
		float top = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
		top		  = fmaxf(top, swap16(top));
		top		  = fmaxf(top, swap32(top)) * c;
		const float m_new = fmaxf(m, top);
		const float base  = m_new == -__builtin_inff() ? 0.0f : m_new; // (no key yet: every weight is 2^-inf)
		if (__builtin_amdgcn_ballot_w64(m_new != m)) {
			const float f = exp2_fast(m - base);
			l *= f;
#pragma unroll
			for (int t = 0; t < DT; ++t) {
				o[t] *= f;
			}
			m = m_new;
		}
		const float shift = weight_bias<CACHE> - base;
		float x[8];
#pragma unroll
		for (int j = 0; j < 8; ++j) {
			x[j] = exp2_fast(fmaf(s[j >> 2][j & 3], c, shift));
			l += x[j];
		}
		vec t[N];
		split8<CACHE, N>(x, t);
#pragma unroll
		for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
			for (int n = N - 1; n >= 0; --n) {
				o[dt] = H::mfma16(d.v[dt], t[n], o[dt]);
			}
		}
	};

	// two steps in turn: one's loads in flight under the other's arithmetic, the page numbers a step ahead of the loads
	step_data d0, d1;
	const int stride = PIECE_UNIT;
	int base		 = p.first_key + wave * STEP;
	load_pages(base, d0);
	load_pages(base + stride, d1);
	if (base < p.end_key) {
		load_step(d0);
	}
	while (base < p.end_key) {
		if (base + stride < p.end_key) {
			load_step(d1);
		}
		compute(d0);
		load_pages(base + 2 * stride, d0);
		base += stride;
		if (base >= p.end_key) {
			break;
		}
		if (base + stride < p.end_key) {
			load_step(d0);
		}
		compute(d1);
		load_pages(base + 2 * stride, d1);
		base += stride;
	}

	// the four waves' results into one: the upper half's into the lower half's, twice
	l += swap16(l);
	l += swap32(l);
#pragma unroll
	for (int upper = WAVES / 2; upper >= 1; upper >>= 1) {
		if (wave >= upper && wave < 2 * upper) {
#pragma unroll
			for (int dt = 0; dt < DT; ++dt) {
				join_o[wave - upper][dt][lane] = o[dt];
			}
			join_ml[wave - upper][0][lane] = m;
			join_ml[wave - upper][1][lane] = l;
		}
		__syncthreads();
		if (wave < upper) {
			const float m2 = join_ml[wave][0][lane], l2 = join_ml[wave][1][lane];
			const float both = fmaxf(m, m2), at = both == -__builtin_inff() ? 0.0f : both;
			const float f1 = exp2_fast(m - at), f2 = exp2_fast(m2 - at);
			l = l * f1 + l2 * f2;
			m = both;
#pragma unroll
			for (int dt = 0; dt < DT; ++dt) {
				const v4f o2 = join_o[wave][dt][lane];
				o[dt]		 = o[dt] * f1 + o2 * f2;
			}
		}
		__syncthreads();
	}
	if (wave != 0) {
		return;
	}
	if (head == 0 && ctile == 0 && lane == 0 && piece == p.first) {
		w.pieces[p.seq] = sequence_pieces{ p.first, p.count };
	}
	if (!there) {
		return;
	}
	if (p.count == 1 && a.prefix_count == 0) {
		const float inv	 = l > 0.0f || l != l ? 1.0f / l : 0.0f;
		const int64_t at = (static_cast<int64_t>(p.seq) * a.q_heads + q_head) * D + 4 * quarter;
#pragma unroll
		for (int dt = 0; dt < DT; ++dt) {
			store_out4<TYPE>(a.out, at + 16 * dt, o[dt][0] * inv, o[dt][1] * inv, o[dt][2] * inv, o[dt][3] * inv);
		}
		return;
	}
	const int64_t to = static_cast<int64_t>(piece) * a.q_heads + q_head;
	if (quarter == 0) {
		w.own_ml[to] = make_float2(m, l);
	}
#pragma unroll
	for (int dt = 0; dt < DT; ++dt) {
		store_out4<NH_F32>(w.own_o, to * D + 4 * quarter + 16 * dt, o[dt][0], o[dt][1], o[dt][2], o[dt][3]);
	}
}

// The pieces of one sequence and query head into one result: 32 (16) lanes hold an output row, eight (sixteen) groups of them take the pieces in turn.
template<int TYPE, int D> __global__ __launch_bounds__(THREADS) void attention_join_kernel(attention_args a, decode_workspace w, int prefix_pieces) {
	constexpr int LANES	 = D / 4;
	constexpr int GROUPS = THREADS / LANES;
	__shared__ float4 join_o[GROUPS][LANES];
	__shared__ float join_ml[GROUPS][2];
	const int seq = blockIdx.x / a.q_heads, q_head = blockIdx.x % a.q_heads;
	const int x = threadIdx.x % LANES, g = threadIdx.x / LANES;
	const int prefix_keys = a.prefix_count << a.cache.page_shift, held = a.batch.width << a.cache.page_shift;
	sequence_pieces own{ 0, 0 };
	if (own_keys(a.batch, prefix_keys, held, seq) > 0) { // (a sequence without any has no piece, and nobody has noted it)
		own = w.pieces[seq];
	}
	if (own.count == 1 && prefix_pieces == 0) {
		return; // written already
	}
	float m = -__builtin_inff(), l = 0.0f;
	float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
	for (int i = g; i < prefix_pieces + own.count; i += GROUPS) {
		const bool shared = i < prefix_pieces;
		const int64_t at  = shared ? (static_cast<int64_t>(i) * a.batch.sequences + seq) * a.q_heads + q_head : static_cast<int64_t>(own.first + i - prefix_pieces) * a.q_heads + q_head;
		const float2 ml	  = shared ? w.prefix_ml[at] : w.own_ml[at];
		const float4 v	  = reinterpret_cast<const float4*>((shared ? w.prefix_o : w.own_o) + at * D)[x];
		const float both = fmaxf(m, ml.x), to = both == -__builtin_inff() ? 0.0f : both;
		const float f1 = exp2_fast(m - to), f2 = exp2_fast(ml.x - to);
		l = l * f1 + ml.y * f2;
		m = both;
		o = make_float4(o.x * f1 + v.x * f2, o.y * f1 + v.y * f2, o.z * f1 + v.z * f2, o.w * f1 + v.w * f2);
	}
	join_o[g][x] = o;
	if (x == 0) {
		join_ml[g][0] = m;
		join_ml[g][1] = l;
	}
	__syncthreads();
	if (g != 0) {
		return;
	}
	for (int i = 1; i < min(GROUPS, prefix_pieces + own.count); ++i) {
		const float m2 = join_ml[i][0], l2 = join_ml[i][1];
		const float4 v	 = join_o[i][x];
		const float both = fmaxf(m, m2), to = both == -__builtin_inff() ? 0.0f : both;
		const float f1 = exp2_fast(m - to), f2 = exp2_fast(m2 - to);
		l = l * f1 + l2 * f2;
		m = both;
		o = make_float4(o.x * f1 + v.x * f2, o.y * f1 + v.y * f2, o.z * f1 + v.z * f2, o.w * f1 + v.w * f2);
	}
	const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f; // no key at all: zeros
	store_out4<TYPE>(a.out, (static_cast<int64_t>(seq) * a.q_heads + q_head) * D + 4 * x, o.x * inv, o.y * inv, o.z * inv, o.w * inv);
}

int64_t attention_decode_workspace(int64_t sequences, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t prefix_keys) {
	decode_workspace w;
	const prefix_cut prefix = plan_prefix(sequences, q_heads / kv_heads, kv_heads, prefix_keys);
	return lay_out(nullptr, sequences, q_heads, head_dim, plan_own(q_heads / kv_heads, kv_heads).units + sequences, prefix.pieces, &w);
}

template<int CACHE, int TYPE, int D> static hipError_t launch_decode(const attention_args& a, hipStream_t s) {
	const int64_t group = a.q_heads / a.cache.kv_heads, sequences = a.batch.sequences;
	const own_cut own		= plan_own(group, a.cache.kv_heads);
	const prefix_cut prefix = plan_prefix(sequences, group, a.cache.kv_heads, static_cast<int64_t>(a.prefix_count) << a.cache.page_shift);
	decode_workspace w;
	(void)lay_out(static_cast<char*>(a.workspace), sequences, a.q_heads, D, own.units + sequences, prefix.pieces, &w);
	if (prefix.pieces > 0) {
		const hipError_t e = launch_attention_prefix(a, CACHE, TYPE, prefix, w.prefix_o, w.prefix_ml, s);
		if (e != hipSuccess) {
			return e;
		}
	}
	const dim3 grid(static_cast<unsigned>((own.units + sequences) * a.cache.kv_heads * own.column_tiles));
	attention_decode_kernel<CACHE, TYPE, D><<<grid, dim3(THREADS), 0, s>>>(a, w, static_cast<int>(own.units), static_cast<int>(own.column_tiles));
	const hipError_t e = hipGetLastError();
	if (e != hipSuccess) {
		return e;
	}
	attention_join_kernel<TYPE, D><<<dim3(static_cast<unsigned>(sequences * a.q_heads)), dim3(THREADS), 0, s>>>(a, w, static_cast<int>(prefix.pieces));
	return hipGetLastError();
}
template<int CACHE, int TYPE> static hipError_t launch_decode(const attention_args& a, hipStream_t s) {
	return a.head_dim == 64 ? launch_decode<CACHE, TYPE, 64>(a, s) : launch_decode<CACHE, TYPE, 128>(a, s);
}

hipError_t launch_attention_decode(const attention_args& a, int cache_type, int type, hipStream_t s) {
	if (cache_type == NH_F16) {
		return type == NH_F32 ? launch_decode<NH_F16, NH_F32>(a, s) : launch_decode<NH_F16, NH_F16>(a, s);
	}
	return type == NH_F32 ? launch_decode<NH_BF16, NH_F32>(a, s) : launch_decode<NH_BF16, NH_BF16>(a, s);
}

} // namespace nh
