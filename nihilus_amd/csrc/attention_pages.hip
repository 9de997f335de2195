// The paged cache from one step to the next (which pages a child keeps, shares, gets and has copied), and its compaction, gfx950.
//
// Who holds a page follows from the page tables and the lengths alone, so nothing is counted between calls: a call marks the held pages
// and takes the rest as free.  Then the pages that have to move are copied, in all layers.  No move's source is another's destination:
// destinations are free pages.  One launch, in which every workgroup works the whole plan out for itself, or, for a cache whose plan does not
// fit in LDS, two.
//
// The plan is a few passes over the tables and one int32 per page of the cache, bound by latency; the copy moves 2 * layers * page bytes per
// page each way and is bound by memory.  Measured: a step of four sequences 6.1 us, of 16 beams that moves 117 MB 29 us (8 TB/s: part
// of it stays in the last-level cache); a compaction of 8 sequences 8.4 us, one that moves 289 MB 122 - 127 us, 4.7 TB/s, the rate of a large copy.
#include "attention_device.h"

#include <algorithm>

namespace nh {

namespace {

constexpr int THREADS = 1024;
constexpr int FREE	  = 0x7FFFFFFF;
constexpr int PER	  = 8; // pages per thread and round of a scan over the cache

struct pages_workspace {
	int32_t* holder; // [pages]  FREE; step: 0 = some child holds it as a full page, i + 1 = child i is the lowest that goes on writing into it.  compact: where it goes
	int32_t* list; // [pages]  free pages (step) or holes (compact), ascending
	int32_t* src; // [moves]
	int32_t* dst;
	int32_t* first; // [children]  rank of the first page given to a child
	int32_t* copied; // [children]  its copy's rank among the copies, -1 without one
	int32_t* moves; // [1]
};
int64_t lay_out(char* base, int64_t pages, int64_t children, pages_workspace* w) {
	int64_t at = 0;
	auto part  = [&](int64_t count) {
		int32_t* p = reinterpret_cast<int32_t*>(base + at);
		at += (count * 4 + 255) / 256 * 256;
		return p;
	};
	w->holder = part(pages);
	w->list	  = part(pages);
	w->src	  = part(std::max(pages, children));
	w->dst	  = part(std::max(pages, children));
	w->first  = part(children);
	w->copied = part(children);
	w->moves  = part(1);
	return at;
}

// What the plan keeps for itself while it runs: in LDS if it is no more than this (a step of 1024 children in a cache of 16384 pages), where no pass over it is a round trip
// to memory (the plan of a step of four sequences 8.7 -> 5.3 us) and where every workgroup can have its own.
constexpr int LDS_WORDS = 2 * 16384 + 4 * 1024;
bool plan_fits_lds(int64_t pages, int64_t children) {
	return std::max(2 * pages + 4 * children, 3 * pages) <= LDS_WORDS; // of a step, of a compaction
}
template<bool LDS> struct words {
	int32_t* p;
	// (in memory: past the vector cache, which does not see what other threads of the workgroup have written or changed by atomics)
	__device__ __forceinline__ int get(int i) const {
		if constexpr (LDS) {
			return p[i];
		} else {
			return __hip_atomic_load(p + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
		}
	}
	__device__ __forceinline__ void put(int i, int v) const {
		if constexpr (LDS) {
			p[i] = v;
		} else {
			__hip_atomic_store(p + i, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
		}
	}
	__device__ __forceinline__ void least(int i, int v) const {
		atomicMin(p + i, v);
	}
};
template<bool LDS> __device__ __forceinline__ void settle() {
	if constexpr (!LDS) {
		wait_stores_acknowledged();
	}
	__syncthreads();
}

// Sum of the threads' values in front of this one, and of all (total).  Every thread of the workgroup calls it.
__device__ __forceinline__ int scan(int v, int& total) {
	__shared__ int sums[THREADS / 64];
	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
	int upto = v;
#pragma unroll
	for (int d = 1; d < 64; d <<= 1) {
		const int other = __shfl_up(upto, d);
		upto += lane >= d ? other : 0;
	}
	if (lane == 63) {
		sums[wave] = upto;
	}
	__syncthreads();
	int before = 0, all = 0;
#pragma unroll
	for (int w = 0; w < THREADS / 64; ++w) {
		before += w < wave ? sums[w] : 0;
		all += sums[w];
	}
	__syncthreads();
	total = all;
	return before + upto - v;
}

struct child {
	const int32_t* row; // of the parent's page table
	int kept, need; // pages that it goes on holding; pages that its new length takes
	int length;
	bool partial; // the last of the kept ones is not full: it will be written into
};
__device__ __forceinline__ child child_of(const pages_args& a, int i) {
	child c{ a.batch.table, 0, 0, 0, false };
	const int p = a.parents[i];
	if (p < 0 || p >= a.batch.sequences) {
		return c;
	}
	const int64_t room = static_cast<int64_t>(a.batch.width) << a.page_shift;
	const int64_t had  = max(int64_t{ 0 }, min(room, static_cast<int64_t>(a.batch.lengths[p])));
	const int64_t now  = max(int64_t{ 0 }, min(room, had + a.grow[i]));
	const int64_t keep = min(had, now), page = int64_t{ 1 } << a.page_shift;
	c.row	  = a.batch.table + static_cast<int64_t>(p) * a.batch.width;
	c.kept	  = static_cast<int>((keep + page - 1) >> a.page_shift);
	c.need	  = static_cast<int>((now + page - 1) >> a.page_shift);
	c.length  = static_cast<int>(now);
	c.partial = (keep & (page - 1)) != 0;
	return c;
}
__device__ __forceinline__ bool in_cache(const pages_args& a, int id) {
	return id >= 0 && id < a.pages;
}
// The listed pages, keys and values of every layer, 8 KiB of one at a time by each team of 256 threads.
constexpr int TEAM		   = 256;
constexpr int COPY_VECTORS = 2; // 16 bytes each, per thread and turn (four: a large compaction 129 us, two: 121)
constexpr int COPY_BYTES   = TEAM * COPY_VECTORS * 16;
template<bool LDS> __device__ __forceinline__ void copy_pages(const pages_args& a, words<LDS> src_pages, words<LDS> dst_pages, int moves, int team, int teams) {
	const int thread	 = threadIdx.x % TEAM;
	const int64_t chunks = (a.page_bytes + COPY_BYTES - 1) / COPY_BYTES;
	const int64_t each	 = 2 * a.layers * chunks, jobs = moves * each;
	for (int64_t job = team; job < jobs; job += teams) {
		const int64_t move = job / each, rest = job % each;
		const int64_t chunk = rest % chunks, layer = rest / chunks >> 1;
		char* pages			= reinterpret_cast<char*>((rest / chunks) & 1 ? a.v : a.k) + layer * a.pages * a.page_bytes;
		const char* src		= pages + src_pages.get(static_cast<int>(move)) * a.page_bytes + chunk * COPY_BYTES;
		char* dst			= pages + dst_pages.get(static_cast<int>(move)) * a.page_bytes + chunk * COPY_BYTES;
		const int64_t left	= a.page_bytes - chunk * COPY_BYTES;
		v4u v[COPY_VECTORS];
#pragma unroll
		for (int i = 0; i < COPY_VECTORS; ++i) {
			const int at = (i * TEAM + thread) * 16;
			if (at < left) {
				v[i] = *reinterpret_cast<const v4u*>(src + at);
			}
		}
#pragma unroll
		for (int i = 0; i < COPY_VECTORS; ++i) {
			const int at = (i * TEAM + thread) * 16;
			if (at < left) {
				*reinterpret_cast<v4u*>(dst + at) = v[i];
			}
		}
	}
}

} // namespace

// LDS: every workgroup works the plan out for itself and copies its part; the first one writes the tables.  Otherwise one workgroup plans.
template<bool LDS> __global__ __launch_bounds__(THREADS) void cache_step_kernel(pages_args a, pages_workspace w) {
	extern __shared__ int32_t shared[];
	const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
	const words<LDS> holder{ LDS ? shared : w.holder }, list{ LDS ? shared + a.pages : w.list };
	int32_t* const for_children = shared + 2 * a.pages;
	const words<LDS> first{ LDS ? for_children : w.first }, copied{ LDS ? for_children + a.children : w.copied };
	const words<LDS> src{ LDS ? for_children + 2 * a.children : w.src }, dst{ LDS ? for_children + 3 * a.children : w.dst };
	const bool writes = blockIdx.x == 0;
	__shared__ int lost, moved; // entries of kept pages that the cache does not have; pages copied
	if (tid == 0) {
		lost = moved = 0;
	}
	for (int p = tid; p < a.pages; p += THREADS) {
		holder.put(p, FREE);
	}
	settle<LDS>();
	for (int i = wave; i < a.children; i += THREADS / 64) {
		const child c = child_of(a, i);
		for (int slot = lane; slot < c.kept; slot += 64) {
			const int id = c.row[slot];
			if (in_cache(a, id)) {
				holder.least(id, c.partial && slot == c.kept - 1 ? i + 1 : 0);
			} else {
				atomicAdd(&lost, 1);
			}
		}
	}
	settle<LDS>();
	// what each child is given, in the children's order
	int given_before = 0, copies_before = 0;
	for (int base = 0; base < a.children; base += THREADS) {
		const int i = base + tid;
		int copy = 0, want = 0;
		if (i < a.children) {
			const child c = child_of(a, i);
			if (c.partial) { // its last page has to be its own
				const int id = c.row[c.kept - 1];
				copy		 = in_cache(a, id) && holder.get(id) != i + 1;
			}
			want = copy + c.need - c.kept;
		}
		int all_wants, all_copies;
		const int rank = given_before + scan(want, all_wants), copy_rank = copies_before + scan(copy, all_copies);
		if (i < a.children) {
			first.put(i, rank);
			copied.put(i, copy ? copy_rank : -1);
		}
		given_before += all_wants;
		copies_before += all_copies;
	}
	const int wanted = given_before;
	// the free pages, ascending, as many as are wanted
	int free_before = 0;
	for (int base = 0; base < a.pages; base += THREADS * PER) {
		const int p0 = base + tid * PER;
		bool is_free[PER];
		int n = 0;
#pragma unroll
		for (int k = 0; k < PER; ++k) {
			is_free[k] = p0 + k < a.pages && holder.get(p0 + k) == FREE;
			n += is_free[k];
		}
		int all;
		int rank = free_before + scan(n, all);
#pragma unroll
		for (int k = 0; k < PER; ++k) {
			if (is_free[k]) {
				if (rank < wanted) {
					list.put(rank, p0 + k);
				}
				++rank;
			}
		}
		free_before += all;
	}
	settle<LDS>();
	const int given = min(wanted, free_before);
	for (int i = wave; i < a.children; i += THREADS / 64) {
		const child c	= child_of(a, i);
		const int rank0 = first.get(i), copy_rank = copied.get(i);
		const int copy	= copy_rank >= 0;
		int32_t* row	= a.new_table + static_cast<int64_t>(i) * a.batch.width;
		for (int slot = lane; slot < a.batch.width; slot += 64) {
			int id = -1;
			if (slot < c.need) {
				const bool own = slot >= c.kept || (copy && slot == c.kept - 1); // a page that is given
				if (own) {
					const int rank = rank0 + (slot >= c.kept ? copy + slot - c.kept : 0);
					id			   = rank < given ? list.get(rank) : -1;
				} else {
					id = in_cache(a, c.row[slot]) ? c.row[slot] : -1;
				}
				if (copy && slot == c.kept - 1 && id >= 0) { // (the copies that can be given are the lowest ranks: the list has no gap)
					src.put(copy_rank, c.row[slot]);
					dst.put(copy_rank, id);
					atomicAdd(&moved, 1);
				}
			}
			if (writes) {
				row[slot] = id;
			}
		}
		if (lane == 0 && writes) {
			a.new_lengths[i] = c.length;
		}
	}
	__syncthreads();
	if (tid == 0 && writes) {
		a.info[0] = a.pages - free_before + given;
		a.info[1] = moved;
		a.info[2] = wanted - given + lost;
		if constexpr (!LDS) {
			w.moves[0] = moved;
		}
	}
	if constexpr (LDS) {
		copy_pages(a, src, dst, moved, blockIdx.x * (THREADS / TEAM) + tid / TEAM, gridDim.x * (THREADS / TEAM));
	}
}

template<bool LDS> __global__ __launch_bounds__(THREADS) void cache_compact_kernel(pages_args a, pages_workspace w) {
	extern __shared__ int32_t shared[];
	const words<LDS> holder{ LDS ? shared : w.holder }, list{ LDS ? shared + a.pages : w.list }, src{ LDS ? shared + 2 * a.pages : w.src };
	const bool writes = blockIdx.x == 0;
	const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
	__shared__ int lost;
	if (tid == 0) {
		lost = 0;
	}
	for (int p = tid; p < a.pages; p += THREADS) {
		holder.put(p, FREE);
	}
	settle<LDS>();
	const int64_t room = static_cast<int64_t>(a.batch.width) << a.page_shift, page = int64_t{ 1 } << a.page_shift;
	auto held_by = [&](int s) {
		return static_cast<int>((max(int64_t{ 0 }, min(room, static_cast<int64_t>(a.batch.lengths[s]))) + page - 1) >> a.page_shift);
	};
	for (int s = wave; s < a.batch.sequences; s += THREADS / 64) {
		const int n = held_by(s);
		for (int slot = lane; slot < n; slot += 64) {
			const int id = a.batch.table[static_cast<int64_t>(s) * a.batch.width + slot];
			if (in_cache(a, id)) {
				holder.put(id, id);
			} else {
				atomicAdd(&lost, 1);
			}
		}
	}
	settle<LDS>();
	int used = 0;
	for (int p = tid; p < a.pages; p += THREADS) {
		used += holder.get(p) != FREE;
	}
	int live;
	(void)scan(used, live);
	int holes_before = 0, movers_before = 0;
	for (int base = 0; base < a.pages; base += THREADS * PER) {
		const int p0 = base + tid * PER;
		int kind[PER]; // 1 a hole in front, 2 a page behind that has to move
		int holes = 0, movers = 0;
#pragma unroll
		for (int k = 0; k < PER; ++k) {
			const int p = p0 + k;
			kind[k]		= 0;
			if (p < a.pages) {
				const bool held = holder.get(p) != FREE;
				kind[k]			= p < live ? (held ? 0 : 1) : held ? 2 : 0;
			}
			holes += kind[k] == 1;
			movers += kind[k] == 2;
		}
		int all_holes, all_movers;
		int hole = holes_before + scan(holes, all_holes), mover = movers_before + scan(movers, all_movers);
#pragma unroll
		for (int k = 0; k < PER; ++k) {
			if (kind[k] == 1) {
				list.put(hole++, p0 + k);
			} else if (kind[k] == 2) {
				src.put(mover++, p0 + k);
			}
		}
		holes_before += all_holes;
		movers_before += all_movers;
	}
	settle<LDS>();
	for (int k = tid; k < movers_before; k += THREADS) { // as many holes as movers
		const int from = src.get(k), to = list.get(k);
		if constexpr (!LDS) {
			w.dst[k] = to;
		}
		holder.put(from, to);
	}
	settle<LDS>();
	for (int s = wave; writes && s < a.batch.sequences; s += THREADS / 64) {
		const int n = held_by(s);
		for (int slot = lane; slot < a.batch.width; slot += 64) {
			const int64_t at = static_cast<int64_t>(s) * a.batch.width + slot;
			const int id	 = slot < n ? a.batch.table[at] : -1;
			a.new_table[at]	 = in_cache(a, id) ? holder.get(id) : -1;
		}
	}
	if (tid == 0 && writes) {
		a.info[0] = live;
		a.info[1] = movers_before;
		a.info[2] = lost;
		if constexpr (!LDS) {
			w.moves[0] = movers_before;
		}
	}
	if constexpr (LDS) {
		copy_pages(a, src, list, movers_before, blockIdx.x * (THREADS / TEAM) + tid / TEAM, gridDim.x * (THREADS / TEAM));
	}
}

// (a cache whose plan does not fit in LDS)
__global__ __launch_bounds__(TEAM) void cache_copy_kernel(pages_args a, pages_workspace w) {
	copy_pages(a, words<false>{ w.src }, words<false>{ w.dst }, w.moves[0], blockIdx.x, gridDim.x);
}

int64_t cache_pages_workspace(int64_t pages, int64_t sequences, int64_t) {
	pages_workspace w;
	return plan_fits_lds(pages, sequences) ? 0 : lay_out(nullptr, pages, sequences, &w);
}

// In one launch if the plan fits in LDS (`words` of it), at most one workgroup per CU; else one workgroup that plans and a launch that copies.
template<typename Kernel> static hipError_t launch(Kernel in_lds, Kernel in_memory, bool lds, int64_t words, int64_t most_moves, const pages_args& a, const pages_workspace& w, hipStream_t s) {
	const int64_t jobs = most_moves * 2 * a.layers * ((a.page_bytes + COPY_BYTES - 1) / COPY_BYTES);
	if (lds) {
		const int64_t workgroups = std::max<int64_t>(1, std::min<int64_t>((jobs + THREADS / TEAM - 1) / (THREADS / TEAM), 256));
		in_lds<<<dim3(static_cast<unsigned>(workgroups)), dim3(THREADS), static_cast<size_t>(words * 4), s>>>(a, w);
		return hipGetLastError();
	}
	in_memory<<<dim3(1), dim3(THREADS), 0, s>>>(a, w);
	const hipError_t e = hipGetLastError();
	if (e != hipSuccess || jobs == 0) {
		return e;
	}
	cache_copy_kernel<<<dim3(static_cast<unsigned>(std::min<int64_t>(jobs, 2048))), dim3(TEAM), 0, s>>>(a, w);
	return hipGetLastError();
}

hipError_t launch_cache_step(const pages_args& a, hipStream_t s) {
	pages_workspace w;
	(void)lay_out(static_cast<char*>(a.workspace), a.pages, a.children, &w);
	return launch(cache_step_kernel<true>, cache_step_kernel<false>, plan_fits_lds(a.pages, a.children), 2 * int64_t{ a.pages } + 4 * int64_t{ a.children }, std::min<int64_t>(a.children, a.pages), a, w, s);
}
hipError_t launch_cache_compact(const pages_args& a, hipStream_t s) {
	pages_workspace w;
	(void)lay_out(static_cast<char*>(a.workspace), a.pages, a.batch.sequences, &w);
	return launch(cache_compact_kernel<true>, cache_compact_kernel<false>, plan_fits_lds(a.pages, a.batch.sequences), 3 * int64_t{ a.pages }, a.pages / 2, a, w, s);
}

} // namespace nh
