/*
 * attention_abi.h -- C ABI of what stands between a block's projections on an MI355X (gfx950): rope and the write into a paged
 * key / value cache, causal attention over it, and the cache's pages from one step to the next.
 *
 * The conventions of q8_0_abi.h hold here too: plain C, device pointers unless a name starts with host_, `stream` a hipStream_t,
 * 0 / negative nh_status / positive hipError_t as the result, no exception.  Calls are asynchronous on their stream, allocate nothing
 * and keep nothing: what a call needs for itself is in the memory that it is given.  That is a workspace, whose contents mean nothing
 * before and after a call, and for attention counters, which must be zero when they are first used and are left zero by every call.  Calls on
 * different streams with workspaces and counters of their own are independent, also while captured into graphs; two calls, or two graphs,
 * that share either must not overlap.
 *
 * In the reference these are nodes of the mega cores whose GPU bodies are empty: rope and the cache write of
 * mega_qkv_prep_and_cache_publish (infra/core_traits.hpp:596-616), k.q, softmax, .v and the head merge of mega_attention_apply
 * (:743-766); the customisation points amd_qkv_epilogue and amd_attention of mega_dispatch.hpp are where a host calls them.  Its cache
 * is fp16 (common/kernel_type_profile_traits.hpp:52-71) and one contiguous slice per sequence; pages are this library's.
 *
 * The cache
 *   K pages  [layers][pages][kv_heads][page_size][head_dim]   a key's values side by side
 *   V pages  [layers][pages][kv_heads][head_dim][page_size]   transposed inside the page
 *   Either way sixteen bytes are eight values along the axis that the matrix instruction adds up (head_dim in q.k, keys in p.v), so both
 *   products take their operands from memory as they lie.  page_size is 16, 32, 64, 128 or 256 tokens, head_dim 64 or 128, values fp16 or bf16.
 * A batch
 *   page_table int32 [sequences][table_width], lengths int32 [sequences], starts int32 [sequences + 1] (or NULL: row i is sequence i's only
 *   one).  Rows starts[b] .. starts[b + 1] - 1 of q (k, v, out) are the last tokens of sequence b, whose length counts them: row r stands
 *   at position lengths[b] - (starts[b + 1] - r).  Key j of a sequence is in page page_table[b][j / page_size] at j % page_size.
 *   Sequences of no rows and of no keys are allowed.  Rows in front of starts[0] and from starts[sequences] on belong to nobody: nothing is read or
 *   written for them.  starts must not descend: if they do, a row gets any result or none and may be written into any place of
 *   the sequences' pages, but nothing else is touched.
 *   The tables are device memory and are not looked at before the launch, so what they hold is checked where it is used: a key whose
 *   page is not one of the cache's (an entry outside [0, pages), a position past the table) does not exist -- it is not written, and
 *   attention leaves it out; a row that has no key at all gives zeros.  What lies in the cache behind a sequence's last key is never
 *   part of a result, whatever it is (infinities, NaN), and an infinite or NaN value of a key is part of the results of those rows that see
 *   the key, in its column, and of no others.
 */
#ifndef NIHILUS_AMD_ATTENTION_ABI_H
#define NIHILUS_AMD_ATTENTION_ABI_H

#include "q8_0_abi.h"

#ifdef __cplusplus
extern "C" {
#endif

/* types of q, k, v, out; a cache is NH_F16 or NH_BF16 */
#define NH_F32 0
#define NH_F16 1
#define NH_BF16 2

typedef struct nh_attn_cache {
	void* k_pages;
	void* v_pages;
	int64_t layers; /* 1 for the calls that take a single layer's pages */
	int64_t pages;
	int64_t kv_heads;
	int64_t page_size;
	int64_t head_dim;
	int32_t type;
} nh_attn_cache;

typedef struct nh_attn_batch {
	const int32_t* page_table;
	const int32_t* lengths;
	const int32_t* starts; /* NULL: one row per sequence */
	int64_t sequences;
	int64_t table_width;
} nh_attn_batch;

/* Rotates q [rows][q_heads][head_dim] into q_out and k [rows][kv_heads][head_dim] into the K pages, and writes v into the V pages.
 *   theta = 2 pi turns[i] position,  (a, b) -> (a cos theta - b sin theta, a sin theta + b cos theta),  i < pairs <= head_dim / 2,
 * (a, b) being values (2i, 2i + 1) of a head if interleaved != 0, else (i, i + pairs); values from 2 pairs on are passed through.
 * turns is fp64: the angle of a far position is reduced to a part of a turn in 64 bits, its sine and cosine and the rotation are
 * fp32, and the result is rounded once.  q_stride, k_stride, v_stride: elements from one row to the next (heads of a row are side by side),
 * multiples of 16 bytes, so that parts of one fused projection can be given; q_out is [rows][q_heads][head_dim] without gaps, may be
 * q itself if q has none, and otherwise has no byte in common with q, k or v (NH_ERR_ARGUMENT).  `type` is that of q, k, v and q_out: NH_F32 or the cache's. */
int nh_attn_append_rope(const nh_attn_cache* host_cache, const nh_attn_batch* host_batch, const void* q, const void* k, const void* v, void* q_out, int type, int64_t rows, int64_t q_heads,
	int64_t q_stride, int64_t k_stride, int64_t v_stride, const double* turns, int64_t pairs, int interleaved, void* stream);

/* out[r] = sum_j softmax_j(scale q[r] . k_j) v_j over the keys j <= position of row r, for every row of every sequence; query head h
 * reads kv head h / (q_heads / kv_heads).  q_heads is a multiple of kv_heads.  starts must not be NULL.  out has no gaps and no byte in
 * common with q (NH_ERR_ARGUMENT), nor with the cache or the tables (not checked).  Scores, scale q.k, are fp32: those above 2^23 have no bits behind the
 * point, and results that hang on them may be anything, also infinite or NaN.
 * type NH_F32: q and the softmax weights go through the 16-bit matrix instructions as sums of two (fp16 cache) or three (bf16) terms,
 * 22 or 24 bits; type = the cache's: q as it is, the weights as two terms where rows are few and rounded once where they are many (a second term
 * would be half as much matrix work again; kernel 2 of nh_attn_debug_prompt_kernel, and a prefix that a decode step goes over apart).  Everything else (products' sums, maxima, sums) is fp32.
 * Memory: nh_attn_prompt_needs says how many bytes (0: many rows need none, and the pointers may be NULL; so fewer rows may need more), 256-byte aligned. */
int nh_attn_prompt_needs(int64_t rows, int64_t sequences, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t* host_workspace_bytes, int64_t* host_counter_bytes);
int nh_attn_prompt(const nh_attn_cache* host_cache, const nh_attn_batch* host_batch, const void* q, void* out, int type, int64_t rows, int64_t q_heads, int64_t q_stride, float scale,
	void* workspace, int64_t workspace_bytes, void* counters, int64_t counter_bytes, void* stream);

/* Which kernel nh_attn_prompt runs for these sizes: 1 the one for few rows (16 at a time, the keys of long sequences over several workgroups), 2 the
 * one for many (128 at a time).  Needs no GPU.  force: 0 lets the sizes decide from now on, 1 or 2 takes
 * that kernel always (and goes over a decode step's shared prefix with each sequence's own keys, or apart), -1 changes nothing; a test hook, process-wide, which anything but -1 is refused for (NH_ERR_ARGUMENT) unless
 * the process has NH_Q8_0_DEBUG_HOOKS=1 in its environment. */
int nh_attn_debug_prompt_kernel(int64_t rows, int64_t sequences, int64_t q_heads, int64_t kv_heads, int force);

/* The same for one row per sequence over all of its keys (starts must be NULL, rows = sequences).  The keys j < prefix_count *
 * page_size of EVERY sequence (as far as its length goes) are those of the pages prefix_pages[0 .. prefix_count): they are read once for the
 * whole batch (where that is faster), and the first prefix_count entries of a page_table row are not looked at by this call.  prefix_count = 0: none shared. */
int nh_attn_decode_needs(int64_t sequences, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t prefix_count, int64_t page_size, int64_t* host_workspace_bytes,
	int64_t* host_counter_bytes);
int nh_attn_decode(const nh_attn_cache* host_cache, const nh_attn_batch* host_batch, const int32_t* prefix_pages, int64_t prefix_count, const void* q, void* out, int type, int64_t q_heads,
	int64_t q_stride, float scale, void* workspace, int64_t workspace_bytes, void* counters, int64_t counter_bytes, void* stream);

/* From one step's sequences to the next one's.  New sequence i (i < children) goes on where sequence parents[i] stands (a number
 * outside [0, sequences): it is empty), longer by grow[i] tokens or, if that is negative, shorter; its length stays within
 * [0, table_width * page_size].  Sequences that no child goes on with are ended, pages that no child holds are free.
 *   - Pages that stay full are shared.  The page that a child will go on writing into must be its own: if several children hold it,
 *     the lowest of them keeps it (unless some child holds it as a full page) and the others get copies.
 *   - Pages that a child needs beyond its parent's are given to it; tokens in them are not written.
 *   - Who holds a page is read from the tables alone: the pages of a shared prefix have to be named in a row that goes on, or they are free.
 *   Free pages are given in ascending order, to the children in theirs, to each its copy first; copies move keys and values of all layers.
 * new_table int32 [children][table_width] (entries past a child's last page are -1), new_lengths int32 [children]; these, info and the workspace have no byte in
 * common with each other, the inputs or the cache (NH_ERR_ARGUMENT).
 * info int32 [3]: pages held afterwards, pages copied, pages that could not be given (too few free) or that the old table did not
 * have; their entries are -1, which the calls above leave out.  Nothing of the inputs changes, so a caller that finds pages missing can end
 * sequences and call again.  starts is not used.  workspace: nh_attn_pages_workspace_bytes(pages, children, table_width) bytes, 0 (and it may
 * be NULL) unless the cache is large. */
int64_t nh_attn_pages_workspace_bytes(int64_t pages, int64_t sequences, int64_t table_width);
int nh_attn_cache_step(const nh_attn_cache* host_cache, const nh_attn_batch* host_batch, const int32_t* parents, const int32_t* grow, int64_t children, int32_t* new_table, int32_t* new_lengths,
	int32_t* info, void* workspace, int64_t workspace_bytes, void* stream);

/* Moves the pages that hold the sequences' tokens to the front (as the tables name them, those of a shared prefix too): with n pages in use, the k-th lowest used page >= n goes to the k-th lowest free
 * page < n, in all layers.  new_table int32 [sequences][table_width] names the pages where they are then (entries past a sequence's
 * last page, and those outside the cache, are -1); info int32 [3]: n, pages moved, entries that were outside the cache.  Pages that
 * were free keep what they held unless something moved there.  Workspace, and what may not lie over what, as above. */
int nh_attn_cache_compact(const nh_attn_cache* host_cache, const nh_attn_batch* host_batch, int32_t* new_table, int32_t* info, void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif
