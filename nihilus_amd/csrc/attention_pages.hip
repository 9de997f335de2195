// The paged cache from one step to the next (which pages a child keeps, shares, gets and has copied), and its compaction, gfx950.
//
// Who holds a page follows from the page tables and the lengths alone, so nothing is counted between calls: a call marks the held pages
// and takes the rest as free.  Two launches each: one workgroup plans (marks, scans, writes the new table and a list of moves), the
// other copies the listed pages, in all layers.  No move's source is another's destination: destinations are free pages.
//
// The plan is a few passes over the tables and one int32 per page of the cache, bound by latency; the copy moves 2 * layers * page bytes per
// page each way and is bound by memory.
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
	int32_t* copied; // [children]  1 if that is a copy, its rank among the copies above
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

// A word that other threads of the workgroup have written or changed by an atomic since this CU last read it: past the vector cache.
__device__ __forceinline__ int fresh(const int32_t* p) {
	return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void put(int32_t* p, int v) {
	__hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
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
// child i has to have its last page copied
__device__ __forceinline__ bool copies(const pages_args& a, const pages_workspace& w, const child& c, int i) {
	if (!c.partial) {
		return false;
	}
	const int id = c.row[c.kept - 1];
	return in_cache(a, id) && fresh(w.holder + id) != i + 1;
}

} // namespace

__global__ __launch_bounds__(THREADS) void cache_step_plan_kernel(pages_args a, pages_workspace w) {
	const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
	__shared__ int lost; // entries of kept pages that the cache does not have
	if (tid == 0) {
		lost = 0;
	}
	for (int p = tid; p < a.pages; p += THREADS) {
		put(w.holder + p, FREE);
	}
	wait_stores_acknowledged();
	__syncthreads();
	for (int i = wave; i < a.children; i += THREADS / 64) {
		const child c = child_of(a, i);
		for (int slot = lane; slot < c.kept; slot += 64) {
			const int id = c.row[slot];
			if (in_cache(a, id)) {
				atomicMin(w.holder + id, c.partial && slot == c.kept - 1 ? i + 1 : 0);
			} else {
				atomicAdd(&lost, 1);
			}
		}
	}
	wait_stores_acknowledged();
	__syncthreads();
	// what each child is given, in the children's order
	int given_before = 0, copies_before = 0;
	for (int base = 0; base < a.children; base += THREADS) {
		const int i = base + tid;
		int copy = 0, want = 0;
		if (i < a.children) {
			const child c = child_of(a, i);
			copy		  = copies(a, w, c, i);
			want		  = copy + c.need - c.kept;
		}
		int all_wants, all_copies;
		const int rank = given_before + scan(want, all_wants), copy_rank = copies_before + scan(copy, all_copies);
		if (i < a.children) {
			put(w.first + i, rank);
			put(w.copied + i, copy ? copy_rank : -1);
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
			is_free[k] = p0 + k < a.pages && fresh(w.holder + p0 + k) == FREE;
			n += is_free[k];
		}
		int all;
		int rank = free_before + scan(n, all);
#pragma unroll
		for (int k = 0; k < PER; ++k) {
			if (is_free[k]) {
				if (rank < wanted) {
					put(w.list + rank, p0 + k);
				}
				++rank;
			}
		}
		free_before += all;
	}
	wait_stores_acknowledged();
	__syncthreads();
	const int given = min(wanted, free_before);
	__shared__ int moved;
	if (tid == 0) {
		moved = 0;
	}
	__syncthreads();
	for (int i = wave; i < a.children; i += THREADS / 64) {
		const child c		= child_of(a, i);
		const int first		= fresh(w.first + i), copy_rank = fresh(w.copied + i);
		const int copy		= copy_rank >= 0;
		int32_t* row		= a.new_table + static_cast<int64_t>(i) * a.batch.width;
		for (int slot = lane; slot < a.batch.width; slot += 64) {
			int id = -1;
			if (slot < c.need) {
				const bool own = slot >= c.kept || (copy && slot == c.kept - 1); // a page that is given
				if (own) {
					const int rank = first + (slot >= c.kept ? copy + slot - c.kept : 0);
					id			   = rank < given ? fresh(w.list + rank) : -1;
				} else {
					id = in_cache(a, c.row[slot]) ? c.row[slot] : -1;
				}
				if (copy && slot == c.kept - 1 && id >= 0) { // (the copies that can be given are the lowest ranks: the list has no gap)
					w.src[copy_rank] = c.row[slot];
					w.dst[copy_rank] = id;
					atomicAdd(&moved, 1);
				}
			}
			row[slot] = id;
		}
		if (lane == 0) {
			a.new_lengths[i] = c.length;
		}
	}
	__syncthreads();
	if (tid == 0) {
		w.moves[0] = moved;
		a.info[0]  = a.pages - free_before + given;
		a.info[1]  = moved;
		a.info[2]  = wanted - given + lost;
	}
}

__global__ __launch_bounds__(THREADS) void cache_compact_plan_kernel(pages_args a, pages_workspace w) {
	const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
	__shared__ int lost;
	if (tid == 0) {
		lost = 0;
	}
	for (int p = tid; p < a.pages; p += THREADS) {
		put(w.holder + p, FREE);
	}
	wait_stores_acknowledged();
	__syncthreads();
	const int64_t room = static_cast<int64_t>(a.batch.width) << a.page_shift, page = int64_t{ 1 } << a.page_shift;
	auto held_by = [&](int s) {
		return static_cast<int>((max(int64_t{ 0 }, min(room, static_cast<int64_t>(a.batch.lengths[s]))) + page - 1) >> a.page_shift);
	};
	for (int s = wave; s < a.batch.sequences; s += THREADS / 64) {
		const int n = held_by(s);
		for (int slot = lane; slot < n; slot += 64) {
			const int id = a.batch.table[static_cast<int64_t>(s) * a.batch.width + slot];
			if (in_cache(a, id)) {
				put(w.holder + id, id);
			} else {
				atomicAdd(&lost, 1);
			}
		}
	}
	wait_stores_acknowledged();
	__syncthreads();
	int used = 0;
	for (int p = tid; p < a.pages; p += THREADS) {
		used += fresh(w.holder + p) != FREE;
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
				const bool held = fresh(w.holder + p) != FREE;
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
				put(w.list + hole++, p0 + k);
			} else if (kind[k] == 2) {
				put(w.src + mover++, p0 + k);
			}
		}
		holes_before += all_holes;
		movers_before += all_movers;
	}
	wait_stores_acknowledged();
	__syncthreads();
	for (int k = tid; k < movers_before; k += THREADS) { // as many holes as movers
		const int from = fresh(w.src + k), to = fresh(w.list + k);
		w.dst[k] = to;
		put(w.holder + from, to);
	}
	wait_stores_acknowledged();
	__syncthreads();
	for (int s = wave; s < a.batch.sequences; s += THREADS / 64) {
		const int n = held_by(s);
		for (int slot = lane; slot < a.batch.width; slot += 64) {
			const int64_t at = static_cast<int64_t>(s) * a.batch.width + slot;
			const int id	 = slot < n ? a.batch.table[at] : -1;
			a.new_table[at]	 = in_cache(a, id) ? fresh(w.holder + id) : -1;
		}
	}
	if (tid == 0) {
		w.moves[0] = movers_before;
		a.info[0]  = live;
		a.info[1]  = movers_before;
		a.info[2]  = lost;
	}
}

// The listed pages, keys and values of every layer, 16 KiB of one at a time.
constexpr int COPY_THREADS = 256;
constexpr int COPY_VECTORS = 4; // 16 bytes each, per thread and turn
constexpr int COPY_BYTES   = COPY_THREADS * COPY_VECTORS * 16;
__global__ __launch_bounds__(COPY_THREADS) void cache_copy_kernel(pages_args a, pages_workspace w) {
	const int64_t chunks = (a.page_bytes + COPY_BYTES - 1) / COPY_BYTES;
	const int64_t each	 = 2 * a.layers * chunks, jobs = w.moves[0] * each;
	for (int64_t job = blockIdx.x; job < jobs; job += gridDim.x) {
		const int64_t move = job / each, rest = job % each;
		const int64_t chunk = rest % chunks, layer = rest / chunks >> 1;
		char* pages			= reinterpret_cast<char*>((rest / chunks) & 1 ? a.v : a.k) + layer * a.pages * a.page_bytes;
		const char* src		= pages + w.src[move] * a.page_bytes + chunk * COPY_BYTES;
		char* dst			= pages + w.dst[move] * a.page_bytes + chunk * COPY_BYTES;
		const int64_t left	= a.page_bytes - chunk * COPY_BYTES;
		v4u v[COPY_VECTORS];
#pragma unroll
		for (int i = 0; i < COPY_VECTORS; ++i) {
			const int at = (i * COPY_THREADS + threadIdx.x) * 16;
			if (at < left) {
				v[i] = *reinterpret_cast<const v4u*>(src + at);
			}
		}
#pragma unroll
		for (int i = 0; i < COPY_VECTORS; ++i) {
			const int at = (i * COPY_THREADS + threadIdx.x) * 16;
			if (at < left) {
				*reinterpret_cast<v4u*>(dst + at) = v[i];
			}
		}
	}
}

int64_t cache_pages_workspace(int64_t pages, int64_t sequences, int64_t) {
	pages_workspace w;
	return lay_out(nullptr, pages, sequences, &w);
}

static hipError_t launch_copy(const pages_args& a, const pages_workspace& w, int64_t most_moves, hipStream_t s) {
	const int64_t jobs = most_moves * 2 * a.layers * ((a.page_bytes + COPY_BYTES - 1) / COPY_BYTES);
	if (jobs == 0) {
		return hipSuccess;
	}
	cache_copy_kernel<<<dim3(static_cast<unsigned>(std::min<int64_t>(jobs, 2048))), dim3(COPY_THREADS), 0, s>>>(a, w);
	return hipGetLastError();
}

hipError_t launch_cache_step(const pages_args& a, hipStream_t s) {
	pages_workspace w;
	(void)lay_out(static_cast<char*>(a.workspace), a.pages, a.children, &w);
	cache_step_plan_kernel<<<dim3(1), dim3(THREADS), 0, s>>>(a, w);
	const hipError_t e = hipGetLastError();
	return e != hipSuccess ? e : launch_copy(a, w, std::min<int64_t>(a.children, a.pages), s);
}
hipError_t launch_cache_compact(const pages_args& a, hipStream_t s) {
	pages_workspace w;
	(void)lay_out(static_cast<char*>(a.workspace), a.pages, a.batch.sequences, &w);
	cache_compact_plan_kernel<<<dim3(1), dim3(THREADS), 0, s>>>(a, w);
	const hipError_t e = hipGetLastError();
	return e != hipSuccess ? e : launch_copy(a, w, a.pages / 2, s);
}

} // namespace nh
