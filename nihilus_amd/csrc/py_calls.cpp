// The calls of a model step on several rows (mul_mat, gemm, gemm_residual, rms_norm_quantize, gate_up_silu) and those between its
// projections (append_rope, attention_prompt, attention_decode, cache_step, cache_compact), and those on int8 matrices with a scale per row, as one native function each, for
// nihilus_amd/q8_0.py, attention.py and i8.py: the checks, the output's allocation, the current stream and the call through the C ABI.
//
// What bounds a small projection is the host.  A launch costs it 2.4 us; the same call from Python through ctypes took 7.9 us ([1024 x 4096]
// against one row): 1.3 us for the ctypes call itself, 1.5 us for each tensor that Python allocates, 2.4 us for checks, sizes and the
// stream, against 0.5 us, 0.6 us and 0.1 us here.  The calls of attention.py, with two structures to fill, took 14 to 18 us.
//
// A function returns the result tensor, or a non-zero status of the library as a number, or None for anything but plain tensors of the
// right kinds and sizes (subclasses, modes that intercept torch calls, wrong shapes, ...): the caller then goes the Python way, which
// also makes the error messages.  Nothing is enqueued before None is returned.
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "nihilus_amd/i8_abi.h"

#include <map>
#include <utility>

namespace {

// the arguments of a call, read one after the other; ok() once all have been
struct args {
	PyObject* const* at;
	Py_ssize_t left;
	bool good;

	args(PyObject* const* a, Py_ssize_t n, Py_ssize_t want) : at(a), left(n), good(n == want && !at::impl::torch_function_mode_enabled() && !c10::impl::TorchDispatchModeTLS::any_modes_set()) {
	}
	const at::Tensor* tensor(at::ScalarType type) {
		PyObject* o = good ? *at++ : nullptr;
		if (!o || !THPVariable_CheckExact(o)) {
			good = false;
			return nullptr;
		}
		const at::Tensor& t = THPVariable_Unpack(o);
		good				= t.defined() && t.is_cuda() && t.scalar_type() == type && t.has_storage() && t.is_contiguous();
		return good ? &t : nullptr;
	}
	const at::Tensor* tensor_or_none(at::ScalarType type) {
		if (good && *at == Py_None) {
			++at;
			return nullptr;
		}
		return tensor(type);
	}
	int64_t integer() {
		PyObject* o = good ? *at++ : nullptr;
		if (!o || !PyLong_CheckExact(o)) {
			good = false;
			return 0;
		}
		int overflow	= 0;
		const int64_t v = PyLong_AsLongLongAndOverflow(o, &overflow);
		good			= overflow == 0;
		return v;
	}
	float number() {
		PyObject* o = good ? *at++ : nullptr;
		if (!o || !PyFloat_CheckExact(o)) {
			good = false;
			return 0.0f;
		}
		return static_cast<float>(PyFloat_AS_DOUBLE(o));
	}
};

const float* floats(const at::Tensor& t) {
	return static_cast<const float*>(t.const_data_ptr());
}
at::Tensor bytes_like(const at::Tensor& t, int64_t n) {
	return at::empty({ n }, t.options().dtype(at::kByte));
}
void* stream() { // the current device's, as nihilus_amd/q8_0.py has it
	return c10::hip::getCurrentHIPStream().stream();
}
// rows of a [M, K] or [K] activation; -1 for any other shape
int64_t rows_of(const at::Tensor& x, int64_t k) {
	if (x.dim() == 1) {
		return x.size(0) == k ? 1 : -1;
	}
	return x.dim() == 2 && x.size(1) == k ? x.size(0) : -1;
}

// runs `call` without the interpreter's lock (a full queue makes a launch wait) and hands its output, or its status, to Python
template<typename Call> PyObject* finish(const at::Tensor& out, Call call) {
	int status;
	Py_BEGIN_ALLOW_THREADS
	status = call();
	Py_END_ALLOW_THREADS
	return status == 0 ? THPVariable_Wrap(out) : PyLong_FromLong(status);
}

// any exception of torch's (an allocation that fails, a tensor without memory): the Python way raises it
template<PyObject* (*F)(args&)> PyObject* guarded(PyObject* const* a, Py_ssize_t n, Py_ssize_t want) {
	try {
		args in(a, n, want);
		if (PyObject* out = in.good ? F(in) : nullptr) {
			return out;
		}
	} catch (const std::exception&) {
	}
	PyErr_Clear();
	Py_RETURN_NONE;
}
template<PyObject* (*F)(args&), int WANT> PyObject* entry(PyObject*, PyObject* const* a, Py_ssize_t n) {
	return guarded<F>(a, n, WANT);
}

// mul_mat(w_tiled, x, n, k, residual or None)
PyObject* mul_mat(args& in) {
	const at::Tensor* w = in.tensor(at::kByte);
	const at::Tensor* x = in.tensor(at::kFloat);
	const int64_t n = in.integer(), k = in.integer();
	const at::Tensor* residual = in.tensor_or_none(at::kFloat);
	const int64_t m			   = in.good ? rows_of(*x, k) : -1;
	if (m < 0 || w->numel() != nh_q8_0_tiled_bytes(n, k) || (residual && residual->numel() != m * n)) {
		return nullptr;
	}
	const int64_t need = nh_q8_0_mul_mat_workspace_bytes(m, k);
	if (need < 0) {
		return nullptr;
	}
	at::Tensor workspace;
	if (need > 0) {
		workspace = bytes_like(*x, need);
	}
	const at::Tensor y = at::empty({ m, n }, x->options());
	const void* wp	   = w->const_data_ptr();
	const float* xp	   = floats(*x);
	const float* rp	   = residual ? floats(*residual) : nullptr;
	float* yp		   = static_cast<float*>(y.mutable_data_ptr());
	void* ws		   = need > 0 ? workspace.mutable_data_ptr() : nullptr;
	void* s			   = stream();
	return finish(y, [&] { return nh_q8_0_mul_mat_scratch(wp, xp, rp, yp, m, n, k, ws, need, s); });
}

// gemm(w_tiled, aq_tiled, m, n, k, residual or None)
PyObject* gemm(args& in) {
	const at::Tensor* w = in.tensor(at::kByte);
	const at::Tensor* a = in.tensor(at::kByte);
	const int64_t m = in.integer(), n = in.integer(), k = in.integer();
	const at::Tensor* residual = in.tensor_or_none(at::kFloat);
	if (!in.good || w->numel() != nh_q8_0_tiled_bytes(n, k) || a->numel() != nh_q8_0_tiled_bytes(m, k) || (residual && residual->numel() != m * n)) {
		return nullptr;
	}
	const at::Tensor c = at::empty({ m, n }, w->options().dtype(at::kFloat));
	const void *wp = w->const_data_ptr(), *ap = a->const_data_ptr();
	const float* rp = residual ? floats(*residual) : nullptr;
	float* cp		= static_cast<float*>(c.mutable_data_ptr());
	void* s			= stream();
	return finish(c, [&] { return residual ? nh_q8_0_gemm_tiled_residual(wp, ap, rp, cp, m, n, k, s) : nh_q8_0_gemm_tiled(wp, ap, cp, m, n, k, s); });
}

// rms_norm_quantize(x, norm_weight, eps), tiled output
PyObject* rms_norm_quantize(args& in) {
	const at::Tensor* x	 = in.tensor(at::kFloat);
	const at::Tensor* nw = in.tensor(at::kFloat);
	const float eps		 = in.number();
	if (!in.good || x->dim() < 1 || x->dim() > 2) {
		return nullptr;
	}
	const int64_t k = x->size(x->dim() - 1), m = x->dim() == 2 ? x->size(0) : 1, size = nh_q8_0_tiled_bytes(m, k);
	if (nw->numel() != k || size < 0) {
		return nullptr;
	}
	const at::Tensor out = bytes_like(*x, size);
	const float *xp = floats(*x), *np = floats(*nw);
	void *op = out.mutable_data_ptr(), *s = stream();
	return finish(out, [&] { return nh_q8_0_rms_norm_quantize_tiled(xp, np, eps, op, m, k, s); });
}

// gate_up_silu(w_gate, w_up, aq_tiled, m, n_ff, k)
PyObject* gate_up_silu(args& in) {
	const at::Tensor* g = in.tensor(at::kByte);
	const at::Tensor* u = in.tensor(at::kByte);
	const at::Tensor* a = in.tensor(at::kByte);
	const int64_t m = in.integer(), n_ff = in.integer(), k = in.integer();
	if (!in.good) {
		return nullptr;
	}
	const int64_t size = nh_q8_0_tiled_bytes(m, n_ff), need = nh_q8_0_gate_up_silu_workspace_bytes(m, n_ff, k);
	if (size < 0 || need < 0) {
		return nullptr;
	}
	const int64_t w_size = nh_q8_0_tiled_bytes(n_ff, k);
	if (size > 0 && (g->numel() < w_size || u->numel() < w_size || a->numel() < nh_q8_0_tiled_bytes(m, k))) {
		return nullptr; // larger buffers than the operands are taken, as by the Python way
	}
	const at::Tensor out = bytes_like(*a, size);
	at::Tensor workspace;
	if (need > 0) {
		workspace = bytes_like(*a, need);
	}
	const void *gp = g->const_data_ptr(), *up = u->const_data_ptr(), *ap = a->const_data_ptr();
	void *op = out.mutable_data_ptr(), *ws = need > 0 ? workspace.mutable_data_ptr() : nullptr, *s = stream();
	return finish(out, [&] { return nh_q8_0_gemm_tiled_gate_up_silu(gp, up, ap, op, ws, need, m, n_ff, k, s); });
}

// ---- attention.py: layouts and meanings as in attention_abi.h ----

// A tensor of any of the types that attention takes; strided ones too.
const at::Tensor* rows_tensor(args& in) {
	PyObject* o = in.good ? *in.at++ : nullptr;
	if (!o || !THPVariable_CheckExact(o)) {
		in.good = false;
		return nullptr;
	}
	const at::Tensor& t = THPVariable_Unpack(o);
	in.good				= t.defined() && t.is_cuda() && t.has_storage() && t.layout() == at::kStrided && !t.is_conj() && !t.is_neg();
	return in.good ? &t : nullptr;
}
int type_of(const at::Tensor& t) {
	return t.scalar_type() == at::kFloat ? NH_F32 : t.scalar_type() == at::kHalf ? NH_F16 : t.scalar_type() == at::kBFloat16 ? NH_BF16 : -1;
}
// The cache of `dims` dimensions (5: all layers, 4: one) and the batch of a call: k_pages, v_pages, page_table, lengths.
struct paged {
	const at::Tensor *k, *v, *table, *lengths;
	nh_attn_cache cache{};
	nh_attn_batch batch{};
	bool good = false;

	// a vector or a table of 32-bit integers on the cache's GPU
	bool ints(const at::Tensor* t, int64_t dim) const {
		return t && t->dim() == dim && t->device() == k->device();
	}
	// rows of the cache's head size, its heads side by side; the elements from one to the next
	bool rows(const at::Tensor* t, int64_t heads, int64_t* stride) const {
		if (!t || t->dim() != 3 || t->size(2) != cache.head_dim || (heads > 0 && t->size(1) != heads) || t->device() != k->device() ||
			(t->scalar_type() != at::kFloat && t->scalar_type() != k->scalar_type()) || t->stride(2) != 1 || (t->size(1) > 1 && t->stride(1) != cache.head_dim)) {
			return false;
		}
		*stride = t->size(0) > 1 ? t->stride(0) : t->size(1) * cache.head_dim;
		return true;
	}
	paged(const at::Tensor* k_, const at::Tensor* v_, const at::Tensor* table_, const at::Tensor* lengths_, int64_t dims) : k(k_), v(v_), table(table_), lengths(lengths_) {
		if (!k || !v || !table || !lengths || k->dim() != dims || v->dim() != dims || !k->is_contiguous() || !v->is_contiguous() || k->scalar_type() != v->scalar_type() || type_of(*k) <= NH_F32 ||
			v->device() != k->device() || !ints(table, 2) || !ints(lengths, 1) || lengths->size(0) != table->size(0)) {
			return;
		}
		for (int64_t d = 0; d < dims; ++d) {
			if (v->size(d) != k->size(d < dims - 2 ? d : 2 * dims - 3 - d)) {
				return;
			}
		}
		if (k->device().index() != c10::hip::current_device()) {
			return; // (the Python way changes devices)
		}
		cache = nh_attn_cache{ k->mutable_data_ptr(), v->mutable_data_ptr(), dims == 5 ? k->size(0) : 1, k->size(dims - 4), k->size(dims - 3), k->size(dims - 2),
			k->size(dims - 1), type_of(*k) };
		batch = nh_attn_batch{ static_cast<const int32_t*>(table->const_data_ptr()), static_cast<const int32_t*>(lengths->const_data_ptr()), nullptr, table->size(0), table->size(1) };
		good  = true;
	}
	bool starts(const at::Tensor* t) {
		if (t && (!ints(t, 1) || t->size(0) != batch.sequences + 1)) {
			return false;
		}
		batch.starts = t ? static_cast<const int32_t*>(t->const_data_ptr()) : nullptr;
		return true;
	}
};
at::Tensor like(const at::Tensor& t) {
	return at::empty(t.sizes(), t.options());
}
at::Tensor ints_like(const at::Tensor& t, at::IntArrayRef sizes) {
	return at::empty(sizes, t.options());
}

// Whether memory that a call takes for itself and gives back to torch's allocator may go to the next call on a stream of the same handle: not under the handle that names
// every thread's own default stream, where that call may be another thread's and waits for nothing.  (The Python way refuses it.)
bool own_memory(void* s) {
	return s != static_cast<void*>(hipStreamPerThread);
}

// Counters of zeros for a call on the current stream s of t's device.  Every call leaves them zero, so the calls of a stream, which run one after the other,
// share theirs.  New ones for a stream that is being captured, whose clearing is captured with the call, and for one that is neither the default stream nor of
// torch's pool (torch numbers such a stream by its handle): its owner may destroy it, and the handle come back.
at::Tensor counters_for(const at::Tensor& t, void* s, int64_t bytes) {
	static auto* kept = new std::map<std::pair<int, void*>, at::Tensor>; // (never destroyed: the interpreter's end is too late to free device memory)
	hipStreamCaptureStatus capturing = hipStreamCaptureStatusNone;
	const bool foreign = s && c10::hip::getCurrentHIPStream().id() == reinterpret_cast<intptr_t>(s);
	const bool plain   = !foreign && hipStreamIsCapturing(static_cast<hipStream_t>(s), &capturing) == hipSuccess && capturing == hipStreamCaptureStatusNone;
	const auto zeros   = [&](int64_t n) { return at::zeros({ n }, t.options().dtype(at::kInt)); };
	if (!plain) {
		return zeros(bytes / 4);
	}
	at::Tensor& mine = (*kept)[{ t.device().index(), s }];
	if (!mine.defined() || mine.numel() * 4 < bytes) {
		mine = zeros(std::max<int64_t>(bytes / 4, 16384));
	}
	return mine;
}

// append_rope(q, k, v, k_pages, v_pages, page_table, lengths, turns, starts or None, interleaved)
PyObject* append_rope(args& in) {
	const at::Tensor *q = rows_tensor(in), *k = rows_tensor(in), *v = rows_tensor(in), *kp = rows_tensor(in), *vp = rows_tensor(in);
	const at::Tensor *table = in.tensor(at::kInt), *lengths = in.tensor(at::kInt), *turns = in.tensor(at::kDouble), *starts = in.tensor_or_none(at::kInt);
	const int64_t interleaved = in.integer();
	if (!in.good) {
		return nullptr;
	}
	paged p(kp, vp, table, lengths, 4);
	int64_t qs, ks, vs;
	if (!p.good || !p.starts(starts) || !p.rows(q, 0, &qs) || !p.rows(k, p.cache.kv_heads, &ks) || !p.rows(v, p.cache.kv_heads, &vs) || k->scalar_type() != q->scalar_type() ||
		v->scalar_type() != q->scalar_type() || k->size(0) != q->size(0) || v->size(0) != q->size(0) || !p.ints(turns, 1)) {
		return nullptr;
	}
	const at::Tensor out = like(*q);
	const void *qp = q->const_data_ptr(), *kd = k->const_data_ptr(), *vd = v->const_data_ptr();
	const double* tp = static_cast<const double*>(turns->const_data_ptr());
	void *op = out.mutable_data_ptr(), *s = stream();
	const int type = type_of(*q);
	const int64_t rows = q->size(0), heads = q->size(1), pairs = turns->size(0);
	return finish(out, [&] { return nh_attn_append_rope(&p.cache, &p.batch, qp, kd, vd, op, type, rows, heads, qs, ks, vs, tp, pairs, interleaved != 0, s); });
}

// attention_prompt(q, k_pages, v_pages, page_table, lengths, starts, scale)
PyObject* attention_prompt(args& in) {
	const at::Tensor *q = rows_tensor(in), *kp = rows_tensor(in), *vp = rows_tensor(in);
	const at::Tensor *table = in.tensor(at::kInt), *lengths = in.tensor(at::kInt), *starts = in.tensor(at::kInt);
	const float scale = in.number();
	if (!in.good) {
		return nullptr;
	}
	paged p(kp, vp, table, lengths, 4);
	int64_t qs;
	if (!p.good || !p.starts(starts) || !p.rows(q, 0, &qs)) {
		return nullptr;
	}
	const int64_t rows = q->size(0), heads = q->size(1);
	int64_t need, counter_need;
	if (nh_attn_prompt_needs(rows, p.batch.sequences, heads, p.cache.kv_heads, p.cache.head_dim, &need, &counter_need) != 0) {
		return nullptr;
	}
	void *s = stream(), *ws = nullptr, *cs = nullptr;
	if (need > 0 && !own_memory(s)) {
		return nullptr;
	}
	const at::Tensor out = like(*q);
	at::Tensor workspace, counters;
	if (need > 0) {
		workspace = bytes_like(*q, need), counters = counters_for(*q, s, counter_need);
		ws = workspace.mutable_data_ptr(), cs = counters.mutable_data_ptr();
	}
	const void* qp = q->const_data_ptr();
	void* op	   = out.mutable_data_ptr();
	const int type = type_of(*q);
	return finish(out, [&] { return nh_attn_prompt(&p.cache, &p.batch, qp, op, type, rows, heads, qs, scale, ws, need, cs, counter_need, s); });
}

// attention_decode(q, k_pages, v_pages, page_table, lengths, prefix_pages or None, scale)
PyObject* attention_decode(args& in) {
	const at::Tensor *q = rows_tensor(in), *kp = rows_tensor(in), *vp = rows_tensor(in);
	const at::Tensor *table = in.tensor(at::kInt), *lengths = in.tensor(at::kInt), *prefix = in.tensor_or_none(at::kInt);
	const float scale = in.number();
	if (!in.good) {
		return nullptr;
	}
	paged p(kp, vp, table, lengths, 4);
	int64_t qs;
	if (!p.good || !p.rows(q, 0, &qs) || q->size(0) != p.batch.sequences || (prefix && !p.ints(prefix, 1))) {
		return nullptr;
	}
	const int64_t heads = q->size(1), count = prefix ? prefix->size(0) : 0;
	int64_t need, counter_need;
	if (nh_attn_decode_needs(p.batch.sequences, heads, p.cache.kv_heads, p.cache.head_dim, count, p.cache.page_size, &need, &counter_need) != 0) {
		return nullptr;
	}
	void* s = stream();
	if (need > 0 && !own_memory(s)) {
		return nullptr;
	}
	const at::Tensor out = like(*q), workspace = bytes_like(*q, need), counters = counters_for(*q, s, counter_need);
	const void* qp	  = q->const_data_ptr();
	const int32_t* pp = count > 0 ? static_cast<const int32_t*>(prefix->const_data_ptr()) : nullptr;
	void *op = out.mutable_data_ptr(), *ws = workspace.mutable_data_ptr(), *cs = counters.mutable_data_ptr();
	const int type = type_of(*q);
	return finish(out, [&] { return nh_attn_decode(&p.cache, &p.batch, pp, count, qp, op, type, heads, qs, scale, ws, need, cs, counter_need, s); });
}

// cache_step(k_pages, v_pages, page_table, lengths, parents, grow): (page_table, lengths, info)
PyObject* cache_step(args& in) {
	const at::Tensor *kp = rows_tensor(in), *vp = rows_tensor(in);
	const at::Tensor *table = in.tensor(at::kInt), *lengths = in.tensor(at::kInt), *parents = in.tensor(at::kInt), *grow = in.tensor(at::kInt);
	if (!in.good) {
		return nullptr;
	}
	paged p(kp, vp, table, lengths, 5);
	if (!p.good || !p.ints(parents, 1) || !p.ints(grow, 1) || grow->size(0) != parents->size(0)) {
		return nullptr;
	}
	const int64_t n = parents->size(0), need = nh_attn_pages_workspace_bytes(p.cache.pages, n, p.batch.table_width);
	void* s = stream();
	if (need < 0 || (need > 0 && !own_memory(s))) {
		return nullptr;
	}
	const at::Tensor new_table = ints_like(*table, { n, p.batch.table_width }), now = ints_like(*table, { n }), info = ints_like(*table, { 3 });
	const at::Tensor workspace = need > 0 ? bytes_like(*table, need) : at::Tensor();
	const auto *pp = static_cast<const int32_t*>(parents->const_data_ptr()), *gp = static_cast<const int32_t*>(grow->const_data_ptr());
	auto *tp = static_cast<int32_t*>(new_table.mutable_data_ptr()), *np = static_cast<int32_t*>(now.mutable_data_ptr()), *ip = static_cast<int32_t*>(info.mutable_data_ptr());
	void* ws = need > 0 ? workspace.mutable_data_ptr() : nullptr;
	PyObject* first = finish(new_table, [&] { return nh_attn_cache_step(&p.cache, &p.batch, pp, gp, n, tp, np, ip, ws, need, s); });
	return first && THPVariable_Check(first) ? Py_BuildValue("NNN", first, THPVariable_Wrap(now), THPVariable_Wrap(info)) : first;
}

// cache_compact(k_pages, v_pages, page_table, lengths): (page_table, info)
PyObject* cache_compact(args& in) {
	const at::Tensor *kp = rows_tensor(in), *vp = rows_tensor(in);
	const at::Tensor *table = in.tensor(at::kInt), *lengths = in.tensor(at::kInt);
	if (!in.good) {
		return nullptr;
	}
	paged p(kp, vp, table, lengths, 5);
	if (!p.good) {
		return nullptr;
	}
	const int64_t need = nh_attn_pages_workspace_bytes(p.cache.pages, p.batch.sequences, p.batch.table_width);
	void* s = stream();
	if (need < 0 || (need > 0 && !own_memory(s))) {
		return nullptr;
	}
	const at::Tensor new_table = like(*table), info = ints_like(*table, { 3 });
	const at::Tensor workspace = need > 0 ? bytes_like(*table, need) : at::Tensor();
	auto *tp = static_cast<int32_t*>(new_table.mutable_data_ptr()), *ip = static_cast<int32_t*>(info.mutable_data_ptr());
	void* ws = need > 0 ? workspace.mutable_data_ptr() : nullptr;
	PyObject* first = finish(new_table, [&] { return nh_attn_cache_compact(&p.cache, &p.batch, tp, ip, ws, need, s); });
	return first && THPVariable_Check(first) ? Py_BuildValue("NN", first, THPVariable_Wrap(info)) : first;
}

// ---- i8.py: layouts and meanings as in i8_abi.h ----

// Rows of activations [rows, k] or [k] on the current GPU, the values of a row side by side.
struct i8_activations {
	const at::Tensor* t;
	int64_t rows = 0, k = 0, stride = 0;
	int type = -1;
	bool good = false;

	explicit i8_activations(args& in) : t(rows_tensor(in)) {
		if (!t || t->dim() < 1 || t->dim() > 2 || (type = type_of(*t)) < 0 || t->device().index() != c10::hip::current_device()) {
			return;
		}
		const bool one = t->dim() == 1;
		rows = one ? 1 : t->size(0), k = t->size(one ? 0 : 1), stride = rows > 1 ? t->stride(0) : k;
		good = (k <= 1 || t->stride(one ? 0 : 1) == 1) && stride >= k;
	}
	const void* data() const {
		return t->const_data_ptr();
	}
};
at::ScalarType scalar_of(int64_t type) {
	return type == NH_F32 ? at::kFloat : type == NH_F16 ? at::kHalf : at::kBFloat16;
}
// fp32 or int32 of this many values, on x's GPU
bool i8_vector(const at::Tensor* t, const at::Tensor& x, int64_t n) {
	return t->dim() == 1 && t->size(0) == n && t->device() == x.device();
}
// w [n][k] and xq [m][k], tiled, on the current GPU (larger buffers than the matrices are taken, as by the Python way)
bool i8_operands(const at::Tensor& w, const at::Tensor& xq, int64_t m, int64_t n, int64_t k) {
	const int64_t w_bytes = nh_i8_tiled_bytes(n, k), x_bytes = nh_i8_tiled_bytes(m, k);
	return w_bytes >= 0 && x_bytes >= 0 && w.numel() >= w_bytes && xq.numel() >= x_bytes && xq.device() == w.device() && w.device().index() == c10::hip::current_device();
}

// i8_quantize(x)
PyObject* i8_quantize(args& in) {
	const i8_activations x(in);
	const int64_t size = x.good ? nh_i8_tiled_bytes(x.rows, x.k) : -1;
	if (size < 0) {
		return nullptr;
	}
	const at::Tensor out = at::empty({ size }, x.t->options().dtype(at::kByte));
	void *op = out.mutable_data_ptr(), *s = stream();
	return finish(out, [&, xp = x.data()] { return nh_i8_quantize(xp, x.type, x.stride, op, x.rows, x.k, s); });
}

// i8_rms_norm_quantize(x, norm_weight, eps)
PyObject* i8_rms_norm_quantize(args& in) {
	const i8_activations x(in);
	const at::Tensor* norm = in.tensor(at::kFloat);
	const float eps		   = in.number();
	const int64_t size	   = in.good && x.good && i8_vector(norm, *x.t, x.k) ? nh_i8_tiled_bytes(x.rows, x.k) : -1;
	if (size < 0) {
		return nullptr;
	}
	const at::Tensor out = at::empty({ size }, x.t->options().dtype(at::kByte));
	void *op = out.mutable_data_ptr(), *s = stream();
	return finish(out, [&, xp = x.data(), np = floats(*norm)] { return nh_i8_rms_norm_quantize(xp, x.type, x.stride, np, eps, op, x.rows, x.k, s); });
}

// i8_silu_mul_quantize(gate, up)
PyObject* i8_silu_mul_quantize(args& in) {
	const i8_activations gate(in), up(in);
	const bool same	   = gate.good && up.good && gate.type == up.type && gate.t->sizes() == up.t->sizes();
	const int64_t size = same ? nh_i8_tiled_bytes(gate.rows, gate.k) : -1;
	if (size < 0) {
		return nullptr;
	}
	const at::Tensor out = at::empty({ size }, gate.t->options().dtype(at::kByte));
	void *op = out.mutable_data_ptr(), *s = stream();
	return finish(out, [&, gp = gate.data(), up_ = up.data()] { return nh_i8_silu_mul_quantize(gp, up_, gate.type, gate.stride, up.stride, op, gate.rows, gate.k, s); });
}

// i8_gemm(w, xq, m, n, k, type, residual or None)
PyObject* i8_gemm(args& in) {
	const at::Tensor *w = in.tensor(at::kByte), *xq = in.tensor(at::kByte);
	const int64_t m = in.integer(), n = in.integer(), k = in.integer(), type = in.integer();
	const at::Tensor* residual = in.good ? in.tensor_or_none(scalar_of(type)) : nullptr;
	if (!in.good || !i8_operands(*w, *xq, m, n, k) || (residual && (residual->dim() != 2 || residual->size(0) != m || residual->size(1) != n || residual->device() != w->device()))) {
		return nullptr;
	}
	const at::Tensor y = at::empty({ m, n }, w->options().dtype(scalar_of(type)));
	const void *wp = w->const_data_ptr(), *xp = xq->const_data_ptr(), *rp = residual ? residual->const_data_ptr() : nullptr;
	void *yp = y.mutable_data_ptr(), *s = stream();
	return finish(y, [&] { return nh_i8_gemm(wp, xp, rp, yp, static_cast<int>(type), m, n, k, s); });
}

// i8_mul_mat(w, x, n, k, residual or None, norm_weight or None, eps)
PyObject* i8_mul_mat(args& in) {
	const at::Tensor* w = in.tensor(at::kByte);
	const i8_activations x(in);
	const int64_t n = in.integer(), k = in.integer();
	if (!in.good || !x.good || x.k != k || w->device() != x.t->device()) {
		return nullptr;
	}
	const at::Tensor *residual = in.tensor_or_none(x.t->scalar_type()), *norm = in.tensor_or_none(at::kFloat);
	const float eps			   = in.number();
	const int64_t bytes = nh_i8_tiled_bytes(n, k), need = nh_i8_mul_mat_workspace_bytes(x.rows, k);
	if (!in.good || bytes < 0 || w->numel() < bytes || need < 0 || (norm && !i8_vector(norm, *x.t, k)) ||
		(residual && (residual->dim() != 2 || residual->size(0) != x.rows || residual->size(1) != n || residual->device() != w->device()))) {
		return nullptr;
	}
	void* s = stream();
	if (need > 0 && !own_memory(s)) {
		return nullptr;
	}
	const at::Tensor y = at::empty({ x.rows, n }, x.t->options()), workspace = need > 0 ? bytes_like(*w, need) : at::Tensor();
	const void *wp = w->const_data_ptr(), *xp = x.data(), *rp = residual ? residual->const_data_ptr() : nullptr;
	const float* np = norm ? floats(*norm) : nullptr;
	void *yp = y.mutable_data_ptr(), *ws = need > 0 ? workspace.mutable_data_ptr() : nullptr;
	return finish(y, [&] { return nh_i8_mul_mat(wp, xp, x.type, x.stride, np, eps, rp, yp, x.rows, n, k, ws, need, s); });
}

// i8_token_losses(w, xq, targets, n, k): (losses, lse)
PyObject* i8_token_losses(args& in) {
	const at::Tensor *w = in.tensor(at::kByte), *xq = in.tensor(at::kByte), *targets = in.tensor(at::kInt);
	const int64_t n = in.integer(), k = in.integer();
	if (!in.good || targets->dim() != 1 || targets->device() != w->device()) {
		return nullptr;
	}
	const int64_t m = targets->size(0), need = nh_i8_token_losses_workspace_bytes(m, n, k);
	void* s = stream();
	if (need < 0 || !i8_operands(*w, *xq, m, n, k) || (need > 0 && !own_memory(s))) {
		return nullptr;
	}
	const at::Tensor losses = at::empty({ m }, w->options().dtype(at::kFloat)), lse = at::empty({ m }, w->options().dtype(at::kFloat)), workspace = bytes_like(*w, need);
	const void *wp = w->const_data_ptr(), *xp = xq->const_data_ptr();
	const int32_t* tp = static_cast<const int32_t*>(targets->const_data_ptr());
	float *lp = static_cast<float*>(losses.mutable_data_ptr()), *ep = static_cast<float*>(lse.mutable_data_ptr());
	void* ws		= workspace.mutable_data_ptr();
	PyObject* first = finish(losses, [&] { return nh_i8_token_losses(wp, xp, tp, lp, ep, m, n, k, ws, need, s); });
	return first && THPVariable_Check(first) ? Py_BuildValue("NN", first, THPVariable_Wrap(lse)) : first;
}

// i8_token_losses_grad(w, xq, targets, losses, lse, n, k, grad or None, type)
PyObject* i8_token_losses_grad(args& in) {
	const at::Tensor *w = in.tensor(at::kByte), *xq = in.tensor(at::kByte), *targets = in.tensor(at::kInt), *losses = in.tensor(at::kFloat), *lse = in.tensor(at::kFloat);
	const int64_t n = in.integer(), k = in.integer();
	const at::Tensor* grad = in.tensor_or_none(at::kFloat);
	const int64_t type	   = in.integer();
	if (!in.good || targets->dim() != 1 || targets->device() != w->device()) {
		return nullptr;
	}
	const int64_t m = targets->size(0), need = nh_i8_token_losses_grad_workspace_bytes(m, n, k, static_cast<int>(type));
	void* s = stream();
	if (need < 0 || !i8_operands(*w, *xq, m, n, k) || !i8_vector(losses, *w, m) || !i8_vector(lse, *w, m) || (grad && !i8_vector(grad, *w, m)) || (need > 0 && !own_memory(s))) {
		return nullptr;
	}
	const at::Tensor dx = at::empty({ m, k }, w->options().dtype(scalar_of(type))), workspace = bytes_like(*w, need);
	const void *wp = w->const_data_ptr(), *xp = xq->const_data_ptr();
	const int32_t* tp = static_cast<const int32_t*>(targets->const_data_ptr());
	const float *lp = floats(*losses), *ep = floats(*lse), *gp = grad ? floats(*grad) : nullptr;
	void *dp = dx.mutable_data_ptr(), *ws = workspace.mutable_data_ptr();
	return finish(dx, [&] { return nh_i8_token_losses_grad(wp, xp, tp, lp, ep, gp, dp, static_cast<int>(type), m, n, k, ws, need, s); });
}

template<PyObject* (*F)(args&), int WANT> constexpr PyMethodDef method(const char* name) {
	return { name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<F, WANT>)), METH_FASTCALL, nullptr };
}
PyMethodDef methods[] = { method<mul_mat, 5>("mul_mat"), method<gemm, 6>("gemm"), method<rms_norm_quantize, 3>("rms_norm_quantize"), method<gate_up_silu, 6>("gate_up_silu"),
	method<append_rope, 10>("append_rope"), method<attention_prompt, 7>("attention_prompt"), method<attention_decode, 7>("attention_decode"), method<cache_step, 6>("cache_step"),
	method<cache_compact, 4>("cache_compact"), method<i8_quantize, 1>("i8_quantize"), method<i8_rms_norm_quantize, 3>("i8_rms_norm_quantize"),
	method<i8_silu_mul_quantize, 2>("i8_silu_mul_quantize"), method<i8_gemm, 7>("i8_gemm"), method<i8_mul_mat, 7>("i8_mul_mat"), method<i8_token_losses, 5>("i8_token_losses"),
	method<i8_token_losses_grad, 9>("i8_token_losses_grad"),
	{ nullptr, nullptr, 0, nullptr } };
PyModuleDef module = { PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr };

} // namespace

PyMODINIT_FUNC PyInit__calls() {
	PyObject* m = PyModule_Create(&module);
	if (m && PyModule_AddStringConstant(m, "built_for", NH_BUILT_FOR) != 0) { // nihilus_amd/build.py
		Py_CLEAR(m);
	}
	return m;
}
