// The per-call host work of the Python entry points in native code: checks, output and scratch allocation, the argument
// block and the call into libaf3_dpa.so.  A small call's kernels run for 5 us; the same work in Python took 13 to 45 us.
//
// Every function takes the plain case of its entry point -- ordinary device tensors of matching types on the current
// device, innermost stride 1 -- and answers None for anything else (and for every malformed call), which sends the caller
// to the Python implementation with its conversions and error messages.  A negative number is an af3_status.
#include <Python.h>

#include <array>
#include <atomic>
#include <cmath>
#include <map>
#include <mutex>
#include <unordered_map>
#include <unordered_set>
#include <vector>

#include <ATen/core/Tensor.h>
#include <ATen/hip/EmptyTensor.h>
#include <ATen/ops/clone.h>
#include <ATen/ops/linear.h>
#include <ATen/ops/matmul.h>
#include <c10/hip/HIPCachingAllocator.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/af3_dpa.h"

extern "C" int64_t af3_dpa_workspace_used(const af3_dpa_params*);   // (api.hip; not part of the ABI)
extern "C" int     af3_dpa_log2_domain(const af3_dpa_params*);            // (likewise)
extern "C" int af3_project_suits(int64_t, int64_t, int64_t);              // (projection.hip, likewise)
extern "C" int af3_grid_project(const void*, const int64_t*, const void*, const void*, float, const void*, const void*, const void*, const void*, const void*, int64_t, int64_t, int32_t, float, void*,
								void*, void*, void*, void*, void*);        // (grid_project.hip, likewise)
extern "C" int af3_project(const void*, const void*, const void*, void*, int64_t, int64_t, int64_t, int32_t, void*);

namespace {

using at::Tensor;

// ---- plain tensors ----------------------------------------------------------------------------------------------------
const Tensor* tensor_of(PyObject* o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

bool on_device(const Tensor& t, int dev) { return t.is_cuda() && t.get_device() == dev; }
bool inner_1(const Tensor& t) { return t.stride(-1) == 1; }
int  dtype_code(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? AF3_BF16 : t.scalar_type() == at::kFloat ? AF3_F32 : -1; }
// the current device when the (first) tensor is on it, -1 otherwise; asks the runtime only about device tensors
int device_of(const Tensor* t) {
	if(!t || !t->is_cuda()) return -1;
	const int dev = (int)c10::hip::current_device();
	return t->get_device() == dev ? dev : -1;
}
void* current_stream(int dev) { return (void*)c10::hip::getCurrentHIPStream((c10::DeviceIndex)dev).stream(); }
Tensor new_tensor(at::IntArrayRef sizes, at::ScalarType type, int dev) {
	return Tensor(at::detail::empty_cuda(sizes, type, at::Device(at::kCUDA, (c10::DeviceIndex)dev), std::nullopt));
}
// scratch of one call: the caching allocator hands the block to later work of the same stream only
at::DataPtr new_scratch(int64_t bytes) { return c10::hip::HIPCachingAllocator::get()->allocate((size_t)bytes); }
PyObject* none() { Py_RETURN_NONE; }
PyObject* wrap(Tensor&& t) { return THPVariable_Wrap(std::move(t)); }

struct without_gil {
	PyThreadState* s = PyEval_SaveThread();
	~without_gil() { PyEval_RestoreThread(s); }
};

// key mask in any of its shapes ([L], [B|1, L], [B|1, 1, 1, L], bool): pointer and batch stride (0: one row for all)
struct key_mask {
	const uint8_t* ptr = nullptr;
	int64_t        stride = 0;
};
bool mask_of(PyObject* o, int64_t B, int64_t L, int dev, key_mask& m) {
	if(o == Py_None) return true;
	const Tensor* t = tensor_of(o);
	if(!t || !on_device(*t, dev) || t->scalar_type() != at::kBool) return false;
	const int64_t d = t->dim();
	if(d != 1 && d != 2 && d != 4) return false;
	if(t->size(-1) != L || !inner_1(*t)) return false;
	if(d == 4 && (t->size(1) != 1 || t->size(2) != 1)) return false;
	if(d > 1 && t->size(0) != 1 && t->size(0) != B) return false;
	m.ptr    = static_cast<const uint8_t*>(t->const_data_ptr());
	m.stride = d > 1 && t->size(0) != 1 ? t->stride(0) : 0;
	return true;
}
bool bias_of(PyObject* o, int64_t H, int64_t L, int dev, const Tensor*& t) {
	t = nullptr;
	if(o == Py_None) return true;
	t = tensor_of(o);
	return t && on_device(*t, dev) && t->dim() == 3 && t->size(0) == H && t->size(1) >= L && t->size(2) >= L && inner_1(*t);
}

void put_strides(int64_t (&dst)[3], const Tensor& t) { dst[0] = t.stride(0), dst[1] = t.stride(1), dst[2] = t.stride(2); }
void put_bias(af3_dpa_params& p, const Tensor& b) {
	p.bias = b.const_data_ptr(), p.bias_stride[0] = b.stride(0), p.bias_stride[1] = b.stride(1), p.bias_dtype = dtype_code(b);
}
af3_dpa_params block(int64_t B, int64_t H, int64_t L, int64_t D, int code, int64_t hint) {
	af3_dpa_params p{};
	p.B = B, p.H = H, p.L = L, p.D = D;
	p.io_dtype = p.out_dtype = p.mma_dtype = code;
	p.softmax_scale = (float)std::pow((double)D, -0.5);
	p.q_descale = p.k_descale = p.v_descale = 1.f;
	p.reserved = (int32_t)hint;
	return p;
}
at::DataPtr workspace_for(af3_dpa_params& p, bool exact_bias) {
	at::DataPtr   ws;
	if(!exact_bias) p.reserved |= 4;
	const int64_t bytes = exact_bias ? 0 : af3_dpa_workspace_used(&p);
	if(bytes > 0) ws = new_scratch(bytes), p.workspace = ws.get(), p.workspace_bytes = bytes;
	return ws;
}
int forward(af3_dpa_params& p, bool exact_bias, int dev) {
	const at::DataPtr ws = workspace_for(p, exact_bias);
	return af3_dpa_forward(&p, current_stream(dev));
}
PyObject* answer(int rc, Tensor&& out) { return rc == AF3_OK ? wrap(std::move(out)) : PyLong_FromLong(rc); }

// ---- matrices derived from weights ------------------------------------------------------------------------------------
// Remembered for as long as their sources are the same live tensors at the same version, address and layout.  The weak
// reference keeps a source's address from being handed to another tensor, so the address alone identifies it.  An entry goes with
// its first source (fused.py hears of that and calls forget_source); past MAX_DERIVED entries all go.  Guarded by the GIL.
constexpr size_t MAX_DERIVED = 1024;
using derived_key = std::array<uintptr_t, 5>;   // what (tag), up to four sources
struct key_hash {
	size_t operator()(const derived_key& k) const {
		size_t h = 0;
		for(uintptr_t v : k) h = (h ^ (size_t)(v >> 4)) * 0x9E3779B97F4A7C15ull + (v & 15);
		return h;
	}
};
struct source {
	c10::weak_intrusive_ptr<c10::TensorImpl> ref;
	const void*      ptr;
	int64_t          version;
	at::ScalarType   type;
	std::vector<int64_t> sizes, strides;
};
struct derived {
	std::vector<source> sources;
	Tensor              value;
};
std::unordered_map<derived_key, derived, key_hash>* g_derived = new std::unordered_map<derived_key, derived, key_hash>();   // (never destroyed: tensors must not be freed after the runtime)

bool make_key(int64_t tag, PyObject* const* o, Py_ssize_t n, derived_key& k) {
	k.fill(0);
	k[0] = (uintptr_t)tag;
	if(n < 1 || n > 4) return false;
	for(Py_ssize_t i = 0; i < n; i++) {
		const Tensor* t = tensor_of(o[i]);
		if(!t || t->is_inference()) return false;
		k[1 + i] = reinterpret_cast<uintptr_t>(t->unsafeGetTensorImpl());
	}
	return true;
}
const Tensor* derived_of(int64_t tag, PyObject* const* o, Py_ssize_t n) {
	derived_key k;
	if(!make_key(tag, o, n, k)) return nullptr;
	const auto it = g_derived->find(k);
	if(it == g_derived->end()) return nullptr;
	for(Py_ssize_t i = 0; i < n; i++) {
		const Tensor& t = *tensor_of(o[i]);
		const source& s = it->second.sources[i];
		if(s.ptr != t.const_data_ptr() || s.version != (int64_t)t._version() || s.type != t.scalar_type() || t.sizes() != s.sizes || t.strides() != s.strides) return nullptr;
	}
	return &it->second.value;
}
// remember(tag, value, source...): True for a new entry, None where it is there already or the tensors cannot be remembered
PyObject* py_remember(PyObject*, PyObject* const* a, Py_ssize_t n) {
	HANDLE_TH_ERRORS
	derived_key   k;
	const Tensor* value = n >= 3 ? tensor_of(a[1]) : nullptr;
	if(!value || !make_key(PyLong_AsLongLong(a[0]), a + 2, n - 2, k)) return none();
	const Tensor* known = derived_of(PyLong_AsLongLong(a[0]), a + 2, n - 2);
	if(known && known->is_same(*value)) return none();
	for(auto it = g_derived->begin(); it != g_derived->end();) {
		bool dead = false;
		for(const source& s : it->second.sources) dead = dead || s.ref.expired();
		it = dead ? g_derived->erase(it) : std::next(it);
	}
	if(g_derived->size() >= MAX_DERIVED) g_derived->clear();
	derived d;
	d.value = *value;
	for(Py_ssize_t i = 2; i < n; i++) {
		const Tensor& t = *tensor_of(a[i]);
		d.sources.push_back(source{c10::weak_intrusive_ptr<c10::TensorImpl>(t.getIntrusivePtr()), t.const_data_ptr(), (int64_t)t._version(), t.scalar_type(), t.sizes().vec(), t.strides().vec()});
	}
	(*g_derived)[k] = std::move(d);
	Py_RETURN_TRUE;
	END_HANDLE_TH_ERRORS
}
// recalls(tag, source...): whether a matrix is remembered for these
PyObject* py_recalls(PyObject*, PyObject* const* a, Py_ssize_t n) {
	HANDLE_TH_ERRORS
	return PyBool_FromLong(n >= 2 && derived_of(PyLong_AsLongLong(a[0]), a + 1, n - 1) != nullptr);
	END_HANDLE_TH_ERRORS
}
// forget_source(address of a source's TensorImpl, as Tensor._cdata gives it)
PyObject* py_forget_source(PyObject*, PyObject* const* a, Py_ssize_t n) {
	const uintptr_t source = n == 1 ? (uintptr_t)PyLong_AsUnsignedLongLong(a[0]) : 0;
	if(PyErr_Occurred()) return nullptr;
	for(auto it = g_derived->begin(); it != g_derived->end();) {
		bool uses = false;
		for(size_t i = 1; i < it->first.size(); i++) uses = uses || it->first[i] == source;
		it = source && uses ? g_derived->erase(it) : std::next(it);
	}
	return none();
}
PyObject* py_forget(PyObject*, PyObject*) {
	g_derived->clear();
	return none();
}
// the tags fused.py remembers its matrices under
enum : int64_t { FUSED_WEIGHT = 1, Q_BIAS_ROW = 2, OUT_PROJ_T = 3, GLU_T = 4 };
int64_t tag_of(int64_t what, int64_t head, int code) { return what | (head << 8) | ((int64_t)code << 40); }

// ---- attention --------------------------------------------------------------------------------------------------------
// attention(q, k, v, mask, bias, kernel hint, exact bias)
PyObject* py_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
	HANDLE_TH_ERRORS
	if(n != 7) return none();
	const Tensor *q = tensor_of(a[0]), *k = tensor_of(a[1]), *v = tensor_of(a[2]), *bias;
	if(!q || !k || !v || q->dim() != 4 || q->numel() == 0) return none();
	const int dev = device_of(q), code = dtype_code(*q);
	if(dev < 0 || code < 0 || k->scalar_type() != q->scalar_type() || v->scalar_type() != q->scalar_type() || k->sizes() != q->sizes() || v->sizes() != q->sizes()) return none();
	if(!on_device(*k, dev) || !on_device(*v, dev) || !inner_1(*q) || !inner_1(*k) || !inner_1(*v)) return none();
	const int64_t B = q->size(0), H = q->size(1), L = q->size(2), D = q->size(3);
	key_mask m;
	if(!mask_of(a[3], B, L, dev, m) || !bias_of(a[4], H, L, dev, bias) || (bias && bias->scalar_type() != q->scalar_type())) return none();
	af3_dpa_params p = block(B, H, L, D, code, PyLong_AsLong(a[5]));
	const bool     exact = a[6] == Py_True;
	Tensor         out;
	int            rc;
	{
		without_gil g;
		out = new_tensor(q->sizes(), q->scalar_type(), dev);
		p.q = q->const_data_ptr(), p.k = k->const_data_ptr(), p.v = v->const_data_ptr(), p.out = out.data_ptr();
		put_strides(p.q_stride, *q), put_strides(p.k_stride, *k), put_strides(p.v_stride, *v), put_strides(p.out_stride, out);
		if(bias) put_bias(p, *bias);
		p.key_mask = m.ptr, p.key_mask_stride_b = m.stride;
		rc = forward(p, exact, dev);
	}
	return answer(rc, std::move(out));
	END_HANDLE_TH_ERRORS
}

// attention_fp8(q, k, v, mask, bias, compensated): quantise (two launches), attend
PyObject* py_attention_fp8(PyObject*, PyObject* const* a, Py_ssize_t n) {
	HANDLE_TH_ERRORS
	if(n != 6) return none();
	const Tensor *q = tensor_of(a[0]), *k = tensor_of(a[1]), *v = tensor_of(a[2]), *bias;
	if(!q || !k || !v || q->dim() != 4 || q->numel() == 0) return none();
	const int dev = device_of(q), code = dtype_code(*q);
	if(dev < 0 || code < 0 || k->scalar_type() != q->scalar_type() || v->scalar_type() != q->scalar_type() || k->sizes() != q->sizes() || v->sizes() != q->sizes()) return none();
	if(!on_device(*k, dev) || !on_device(*v, dev) || !q->is_contiguous() || !k->is_contiguous() || !v->is_contiguous()) return none();
	const int64_t B = q->size(0), H = q->size(1), L = q->size(2), D = q->size(3);
	key_mask m;
	if(D % 4 != 0 || !mask_of(a[3], B, L, dev, m) || !bias_of(a[4], H, L, dev, bias) || (bias && bias->scalar_type() != at::kBFloat16)) return none();
	const bool comp = a[5] == Py_True;
	Tensor     out;
	int        rc;
	{
		without_gil g;
		out = new_tensor(q->sizes(), q->scalar_type(), dev);
		// one block: q8, k8, their residuals, v8t (rows padded to 16 keys), the quantiser's floats
		const int64_t each = (q->numel() + 255) & ~255ll, lpad = (L + 15) / 16 * 16, vt = (B * H * D * lpad + 255) & ~255ll;
		at::DataPtr   mem  = new_scratch((comp ? 4 : 2) * each + vt + 256 + AF3_QKV_SCRATCH_FLOATS * 4);
		uint8_t*      at8  = static_cast<uint8_t*>(mem.get());
		uint8_t *q8 = at8, *k8 = q8 + each, *qlo = comp ? k8 + each : nullptr, *klo = comp ? qlo + each : nullptr, *v8 = k8 + (comp ? 3 : 1) * each;
		float *descales = reinterpret_cast<float*>(v8 + vt), *scratch = descales + 64;
		rc = af3_quantize_qkv_fp8_e4m3(q->const_data_ptr(), k->const_data_ptr(), v->const_data_ptr(), code, B, H, L, D, (float)std::pow((double)D, -0.5), q8, k8, v8, lpad, qlo, klo, descales, scratch,
									   current_stream(dev));
		if(rc == AF3_OK) {
			af3_dpa_params p = block(B, H, L, D, AF3_FP8_E4M3, 0);
			p.softmax_scale = 1.f, p.out_dtype = code;
			p.q = q8, p.k = k8, p.v = v8, p.q_lo = qlo, p.k_lo = klo, p.out = out.data_ptr(), p.device_descales = descales;
			put_strides(p.q_stride, *q), put_strides(p.k_stride, *q), put_strides(p.out_stride, out);
			p.v_stride[0] = H * D * lpad, p.v_stride[1] = D * lpad, p.v_stride[2] = lpad;
			if(bias) put_bias(p, *bias);
			p.key_mask = m.ptr, p.key_mask_stride_b = m.stride;
			rc = af3_dpa_forward(&p, current_stream(dev));
		}
	}
	return answer(rc, std::move(out));
	END_HANDLE_TH_ERRORS
}

// the attention launch on the projections y [B*N, 4C] -- per token and head (k | v | q | gate) -- into out [B, N, C]
int attend(const Tensor& y, int64_t B, int64_t N, int64_t head, const key_mask& m, const Tensor* bias, Tensor& out, int64_t hint, bool exact, int dev) {
	const int64_t C = y.size(1) / 4, K = C / head, esz = (int64_t)y.element_size();
	af3_dpa_params p = block(B, head, N, K, dtype_code(y), hint);
	const auto* base = static_cast<const uint8_t*>(y.const_data_ptr());
	p.k = base, p.v = base + K * esz, p.q = base + 2 * K * esz, p.gate = base + 3 * K * esz, p.out = out.data_ptr();
	const int64_t st[3] = {N * 4 * C, 4 * K, 4 * C}, so[3] = {N * C, K, C};
	for(int i = 0; i < 3; i++) p.q_stride[i] = p.k_stride[i] = p.v_stride[i] = p.gate_stride[i] = st[i], p.out_stride[i] = so[i];
	p.bias_dtype = p.io_dtype;
	if(bias) put_bias(p, *bias);
	p.key_mask = m.ptr, p.key_mask_stride_b = m.stride;
	return forward(p, exact, dev);
}

// rows of x [.., C] times the fused projection weight [4C, C], plus the row: this library's kernel where it suits, a library GEMM otherwise
Tensor project(const Tensor& x, int64_t M, const Tensor& weight, const Tensor* row, int dev, int& rc) {
	const int64_t K = weight.size(1), N = weight.size(0);
	rc = AF3_OK;
	if(x.scalar_type() == at::kBFloat16 && weight.is_contiguous() && af3_project_suits(M, N, K)) {
		const Tensor rows = reinterpret_cast<uintptr_t>(x.const_data_ptr()) % 16 == 0 ? x : x.clone();
		Tensor       y    = new_tensor({M, N}, at::kBFloat16, dev);
		rc = af3_project(rows.const_data_ptr(), weight.const_data_ptr(), row ? row->const_data_ptr() : nullptr, y.data_ptr(), M, N, K, 0, current_stream(dev));
		return y;
	}
	return at::linear(x.dim() == 2 ? x : x.reshape({M, K}), weight, row ? *row : Tensor());
}

// self_attention(x [N, C] or [S, N, C], mask, bias, wq, wk, wv, wg, q_bias, head, kernel hint, exact bias)
PyObject* py_self_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
	HANDLE_TH_ERRORS
	if(n != 11) return none();
	const Tensor *x = tensor_of(a[0]), *bias;
	const int64_t head = PyLong_AsLongLong(a[8]);
	const int     dev = device_of(x);
	if(dev < 0 || (x->dim() != 2 && x->dim() != 3) || !x->is_contiguous() || x->numel() == 0 || head < 1) return none();
	const int     code = dtype_code(*x);
	const int64_t C = x->size(-1), N = x->size(-2), S = x->dim() == 3 ? x->size(0) : 1;
	key_mask      m;
	if(code < 0 || C % head != 0 || !mask_of(a[1], S, N, dev, m) || !bias_of(a[2], head, N, dev, bias) || (bias && bias->scalar_type() != x->scalar_type())) return none();
	// (both were derived from checked weights; a call with other ones finds nothing here)
	const Tensor* w  = derived_of(tag_of(FUSED_WEIGHT, head, code), a + 3, 4);
	const Tensor* qb = derived_of(tag_of(Q_BIAS_ROW, head, code), a + 7, 1);
	if(!w || !qb || w->size(1) != C || qb->size(0) != 4 * C || !on_device(*w, dev) || !on_device(*qb, dev)) return none();
	const Tensor weight = *w, row = *qb;
	const int64_t hint = PyLong_AsLongLong(a[9]);
	const bool    exact = a[10] == Py_True;
	Tensor out;
	int    rc;
	{
		without_gil g;
		const Tensor y = project(*x, S * N, weight, &row, dev, rc);
		if(rc != AF3_OK) {
		} else if(y.scalar_type() != x->scalar_type() || !y.is_contiguous()) rc = 1;  // (autocast)
		else {
			out = new_tensor(x->sizes(), x->scalar_type(), dev);
			rc  = attend(y, S, N, head, m, bias, out, hint, exact, dev);
		}
	}
	return rc == 1 ? none() : answer(rc, std::move(out));
	END_HANDLE_TH_ERRORS
}

// ---- grid attention ---------------------------------------------------------------------------------------------------
// The one-kernel form into `out` [B, N, C]: 0, an af3_status, or 1 where the library does not take the shape.
int grid_kernel(const Tensor& pair, const key_mask& m, const Tensor* bias, const Tensor* const (&ws)[4], int64_t head, Tensor& out, int dev) {
	af3_grid_attention_params g{};
	const int64_t B = pair.size(0), N = pair.size(1), C = pair.size(2);
	g.pair = pair.const_data_ptr(), g.pair_stride[0] = pair.stride(0), g.pair_stride[1] = pair.stride(1);
	g.q_proj = ws[0]->const_data_ptr(), g.k_proj = ws[1]->const_data_ptr(), g.v_proj = ws[2]->const_data_ptr(), g.gating_query = ws[3]->const_data_ptr();
	g.B = B, g.N = N, g.C = C, g.head = head, g.dtype = dtype_code(pair);
	if(bias) g.bias = bias->const_data_ptr(), g.bias_stride[0] = bias->stride(0), g.bias_stride[1] = bias->stride(1), g.bias_dtype = dtype_code(*bias);
	g.key_mask = m.ptr, g.key_mask_stride_b = m.stride;
	out   = new_tensor({B, N, C}, pair.scalar_type(), dev);
	g.out = out.data_ptr(), g.out_stride[0] = N * C, g.out_stride[1] = C;
	if(!af3_grid_attention_supported(&g)) return 1;
	at::DataPtr   mem;
	const int64_t bytes = af3_grid_attention_workspace_bytes(&g);
	if(bytes > 0) mem = new_scratch(bytes), g.workspace = mem.get(), g.workspace_bytes = bytes;
	return af3_grid_attention_forward(&g, current_stream(dev));
}
bool grid_weights(PyObject* const* o, const Tensor& pair, int64_t head, int dev, const Tensor* (&ws)[4]) {
	const int64_t C = pair.size(2);
	for(int i = 0; i < 4; i++) {
		ws[i] = tensor_of(o[i]);
		if(!ws[i] || !on_device(*ws[i], dev) || ws[i]->scalar_type() != pair.scalar_type() || ws[i]->dim() != 2 || ws[i]->size(0) != C || ws[i]->size(1) != C || !ws[i]->is_contiguous()) return false;
	}
	return head > 0 && C % head == 0;
}

// grid_kernel(pair, mask, bias, wq, wk, wv, wg, head)
PyObject* py_grid_kernel(PyObject*, PyObject* const* a, Py_ssize_t n) {
	HANDLE_TH_ERRORS
	if(n != 8) return none();
	const Tensor *pair = tensor_of(a[0]), *bias, *ws[4];
	const int64_t head = PyLong_AsLongLong(a[7]);
	const int     dev = device_of(pair);
	key_mask      m;
	if(dev < 0 || pair->dim() != 3 || pair->numel() == 0 || dtype_code(*pair) < 0 || !inner_1(*pair)) return none();
	if(!grid_weights(a + 3, *pair, head, dev, ws) || !mask_of(a[1], pair->size(0), pair->size(1), dev, m) || !bias_of(a[2], head, pair->size(1), dev, bias) || (bias && dtype_code(*bias) < 0)) return none();
	Tensor out;
	int    rc;
	{
		without_gil g;
		rc = grid_kernel(*pair, m, bias, ws, head, out, dev);
	}
	return rc == 1 ? none() : answer(rc, std::move(out));
	END_HANDLE_TH_ERRORS
}

// shapes for which af3_linear beats the library GEMM (measured): bfloat16, 64 or 128 input channels, at most 128 outputs
bool narrow(const Tensor& rows, int64_t n_out) {
	return rows.scalar_type() == at::kBFloat16 && (rows.size(-1) == 64 || rows.size(-1) == 128) && n_out % 32 == 0 && n_out <= 128 && n_out > 0 && rows.numel() > 0 && rows.is_contiguous() &&
		   reinterpret_cast<uintptr_t>(rows.const_data_ptr()) % 16 == 0;
}
int narrow_linear(const Tensor& rows, const Tensor& weight, Tensor& out, int dev) {
	const int64_t K = rows.size(-1), M = rows.numel() / K, N = weight.size(0);
	auto sizes = rows.sizes().vec();
	sizes.back() = N;
	out = new_tensor(sizes, rows.scalar_type(), dev);
	return af3_linear(rows.const_data_ptr(), weight.const_data_ptr(), out.data_ptr(), M, K, N, AF3_BF16, current_stream(dev));
}

// out_projection(rows [.., C], out_proj [C, C] = weight^T)
PyObject* py_out_projection(PyObject*, PyObject* const* a, Py_ssize_t n) {
	HANDLE_TH_ERRORS
	if(n != 2) return none();
	const Tensor *rows = tensor_of(a[0]), *wt = derived_of(OUT_PROJ_T, a + 1, 1);
	const int     dev = device_of(rows);
	if(dev < 0 || !wt || !on_device(*wt, dev) || wt->scalar_type() != rows->scalar_type() || wt->size(1) != rows->size(-1) || !narrow(*rows, wt->size(0))) return none();
	const Tensor weight = *wt;
	Tensor       out;
	int          rc;
	{
		without_gil g;
		rc = narrow_linear(*rows, weight, out, dev);
	}
	return answer(rc, std::move(out));
	END_HANDLE_TH_ERRORS
}

// linear(x [.., K], weight [N, K])
PyObject* py_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
	HANDLE_TH_ERRORS
	if(n != 2) return none();
	const Tensor *x = tensor_of(a[0]), *w = tensor_of(a[1]);
	const int     dev = device_of(x);
	if(dev < 0 || !w || x->dim() < 1 || w->dim() != 2 || !on_device(*w, dev) || w->scalar_type() != x->scalar_type() || w->size(1) != x->size(-1) || !w->is_contiguous() ||
	   !narrow(*x, w->size(0)))
		return none();
	Tensor out;
	int    rc;
	{
		without_gil g;
		rc = narrow_linear(*x, *w, out, dev);
	}
	return answer(rc, std::move(out));
	END_HANDLE_TH_ERRORS
}

// ---- LayerNorm + pair bias ----------------------------------------------------------------------------------------------
struct ln_args {
	const Tensor *pair, *gamma, *beta, *proj;
	float         eps;
};
bool ln_of(PyObject* const* a, int& dev, ln_args& r) {   // a: pair, ln_weight, ln_bias, eps, proj_weight
	r = {tensor_of(a[0]), tensor_of(a[1]), tensor_of(a[2]), tensor_of(a[4]), 0.f};
	dev = device_of(r.pair);
	if(dev < 0 || !r.gamma || !r.beta || !r.proj || r.pair->dim() != 3 || r.proj->dim() != 2 || r.pair->numel() == 0 || dtype_code(*r.pair) < 0 || !inner_1(*r.pair)) return false;
	const int64_t C = r.pair->size(2), head = r.proj->size(0);
	if(r.proj->size(1) != C || r.gamma->numel() != C || r.beta->numel() != C || C > 2048 || head < 1 || head > 64 || (2 + head) * C * 4 > 160 * 1024 - 1024) return false;
	for(const Tensor* t : {r.pair, r.gamma, r.beta, r.proj})
		if(!on_device(*t, dev) || t->scalar_type() != r.pair->scalar_type() || (t != r.pair && !t->is_contiguous())) return false;
	const double eps = PyFloat_AsDouble(a[3]);
	if(eps == -1.0 && PyErr_Occurred()) {
		PyErr_Clear();
		return false;
	}
	r.eps = (float)eps;
	return true;
}
int ln_pair_bias(const ln_args& r, Tensor& normed, Tensor& bias, int dev) {
	const int64_t n_i = r.pair->size(0), n_j = r.pair->size(1), C = r.pair->size(2), head = r.proj->size(0);
	normed = new_tensor({n_i, n_j, C}, r.pair->scalar_type(), dev);
	bias   = new_tensor({head, n_i, n_j}, r.pair->scalar_type(), dev);
	const int64_t ps[2] = {r.pair->stride(0), r.pair->stride(1)}, bs[2] = {n_i * n_j, n_j};
	return af3_layernorm_pair_bias(r.pair->const_data_ptr(), ps, r.gamma->const_data_ptr(), r.beta->const_data_ptr(), r.eps, r.proj->const_data_ptr(), normed.data_ptr(), bias.data_ptr(), bs, n_i, n_j, C,
								   head, dtype_code(*r.pair), current_stream(dev));
}

// layernorm_pair_bias(pair, ln_weight, ln_bias, eps, proj_weight)
PyObject* py_layernorm_pair_bias(PyObject*, PyObject* const* a, Py_ssize_t n) {
	HANDLE_TH_ERRORS
	ln_args   r;
	int       dev = -1;
	if(n != 5 || !ln_of(a, dev, r)) return none();
	Tensor normed, bias;
	int    rc;
	{
		without_gil g;
		rc = ln_pair_bias(r, normed, bias, dev);
	}
	if(rc != AF3_OK) return PyLong_FromLong(rc);
	PyObject *x = wrap(std::move(normed)), *y = x ? wrap(std::move(bias)) : nullptr;
	if(!y) {
		Py_XDECREF(x);
		return nullptr;
	}
	PyObject* both = PyTuple_Pack(2, x, y);
	Py_DECREF(x), Py_DECREF(y);
	return both;
	END_HANDLE_TH_ERRORS
}

// LayerNorm, pair bias and projections in one kernel (128 channels in 4 heads, bfloat16), then the attention launch on q, k, v and the
// gate [B, 4, N, 32] and the output projection.
bool grid_projected_ok(const ln_args& r, const Tensor* const (&ws)[4]) {
	const auto odd = [](const Tensor* t, int to) { return reinterpret_cast<uintptr_t>(t->const_data_ptr()) % to != 0; };
	return r.pair->size(2) == 128 && r.proj->size(0) == 4 && r.pair->scalar_type() == at::kBFloat16 && r.pair->stride(0) % 8 == 0 && r.pair->stride(1) % 8 == 0 && !odd(r.pair, 16) &&
		   !odd(r.gamma, 16) && !odd(r.beta, 16) && !odd(r.proj, 16) && !odd(ws[0], 4) && !odd(ws[1], 4) && !odd(ws[2], 4) && !odd(ws[3], 4);
}
// Where the memory for q, k, v and the gate of the whole call is not there, they go in slabs of batch rows of at most 256 MB, after a
// pass over the whole pair tensor for the bias, which every slab needs (N = 640 414 -> 488 us, 1024 1316 -> 1450).
constexpr int64_t GRID_SLAB_BYTES = (int64_t)256 << 20;
int grid_projected_rows(const ln_args& r, const key_mask& m, const Tensor* const (&ws)[4], bool turned, int64_t hint, bool exact, const Tensor& out_weight, int64_t rows, Tensor& out, int dev) {
	const int64_t n_i = r.pair->size(0), n_j = r.pair->size(1), B = turned ? n_j : n_i, N = turned ? n_i : n_j, each = rows * N * 128;
	const bool    whole = rows == B;
	at::DataPtr   mem = new_scratch((4 * each + 4 * n_i * n_j) * 2), rows_out = new_scratch(each * 2);
	auto* const     q = static_cast<uint16_t*>(mem.get());
	uint16_t *const k = q + each, *const v = k + each, *const gate = v + each, *const bias = gate + each;
	if(!whole) out = new_tensor({B, N, 128}, at::kBFloat16, dev);
	const int64_t ps[2] = {r.pair->stride(0), r.pair->stride(1)};
	const auto project_rows = [&](int64_t b0, int64_t count, float q_scale, bool with_rows, bool with_bias) {
		const auto* x = static_cast<const uint16_t*>(r.pair->const_data_ptr()) + b0 * ps[turned ? 1 : 0];
		return af3_grid_project(x, ps, r.gamma->const_data_ptr(), r.beta->const_data_ptr(), r.eps, r.proj->const_data_ptr(), ws[0]->const_data_ptr(), ws[1]->const_data_ptr(), ws[2]->const_data_ptr(),
								ws[3]->const_data_ptr(), turned ? N : count, turned ? count : N, turned, q_scale, with_rows ? q : nullptr, with_rows ? k : nullptr, with_rows ? v : nullptr,
								with_rows ? gate : nullptr, with_bias ? bias : nullptr, current_stream(dev));
	};
	int rc = whole ? AF3_OK : project_rows(0, B, 1.f, false, true);
	for(int64_t b0 = 0; b0 < B && rc == AF3_OK; b0 += rows) {
		const int64_t  count = B - b0 < rows ? B - b0 : rows;
		af3_dpa_params p = block(count, 4, N, 32, AF3_BF16, hint);
		p.q = q, p.k = k, p.v = v, p.gate = gate, p.out = rows_out.get(), p.bias = bias;
		const int64_t st[3] = {4 * N * 32, N * 32, 32}, so[3] = {N * 128, 32, 128};
		for(int i = 0; i < 3; i++) p.q_stride[i] = p.k_stride[i] = p.v_stride[i] = p.gate_stride[i] = st[i], p.out_stride[i] = so[i];
		p.bias_stride[0] = n_i * n_j, p.bias_stride[1] = n_j, p.bias_dtype = AF3_BF16;
		p.key_mask = m.ptr ? m.ptr + b0 * m.stride : nullptr, p.key_mask_stride_b = m.stride;
		{
			const at::DataPtr work = workspace_for(p, exact);
			// The whole scale of the logits goes into q where it is projected, in fp32: one rounding.  What is left for the attention
			// kernel is 1 in its own units (a product with it gives the same bits back).
			const float log2e = 1.4426950408889634f, q_scale = af3_dpa_log2_domain(&p) ? p.softmax_scale * log2e : p.softmax_scale;
			p.softmax_scale = q_scale == p.softmax_scale ? 1.f : 1.f / log2e;
			rc = project_rows(b0, count, q_scale, true, whole);
			if(rc == AF3_OK) rc = af3_dpa_forward(&p, current_stream(dev));
		}
		if(rc != AF3_OK) break;
		if(whole) mem = at::DataPtr(), out = new_tensor({B, N, 128}, at::kBFloat16, dev);   // (the result may take the place of what is no longer needed)
		rc = af3_linear(rows_out.get(), out_weight.const_data_ptr(), static_cast<uint16_t*>(out.data_ptr()) + b0 * N * 128, count * N, 128, out_weight.size(0), AF3_BF16, current_stream(dev));
	}
	return rc;
}
int grid_projected(const ln_args& r, const key_mask& m, const Tensor* const (&ws)[4], bool turned, int64_t hint, bool exact, const Tensor& out_weight, Tensor& out, int dev) {
	const int64_t B = r.pair->size(turned ? 1 : 0), N = r.pair->size(turned ? 0 : 1), fit = GRID_SLAB_BYTES / (N * 1024) / 32 * 32;
	const int64_t rows = fit < 32 ? 32 : fit;
	if(rows < B) {
		try {
			return grid_projected_rows(r, m, ws, turned, hint, exact, out_weight, B, out, dev);
		} catch(const c10::OutOfMemoryError&) {
		}
	}
	return grid_projected_rows(r, m, ws, turned, hint, exact, out_weight, rows < B ? rows : B, out, dev);
}

// grid_block(pair, ln_weight, ln_bias, eps, proj_weight, mask, wq, wk, wv, wg, out_proj, head, transpose, least (batch row, head) pairs of
// the one-kernel form, kernel hint, exact bias): the whole block of GridSelfAttentionCpp.forward
PyObject* py_grid_block(PyObject*, PyObject* const* a, Py_ssize_t n) {
	HANDLE_TH_ERRORS
	ln_args       r;
	int           dev = -1;
	const Tensor* ws[4];
	key_mask      m;
	if(n != 16 || !ln_of(a, dev, r)) return none();
	const int64_t head = PyLong_AsLongLong(a[11]), least = PyLong_AsLongLong(a[13]), hint = PyLong_AsLongLong(a[14]);
	const bool    turned = a[12] == Py_True, exact = a[15] == Py_True;
	const int64_t B = r.pair->size(turned ? 1 : 0), N = r.pair->size(turned ? 0 : 1), C = r.pair->size(2);
	// (the closing projection is af3_linear: 64 or 128 channels in bfloat16)
	if(B != N || r.pair->scalar_type() != at::kBFloat16 || (C != 64 && C != 128) || r.proj->size(0) != head || !grid_weights(a + 6, *r.pair, head, dev, ws) || !mask_of(a[5], B, N, dev, m)) return none();
	const Tensor* wt = derived_of(OUT_PROJ_T, a + 10, 1);
	const Tensor* wf = derived_of(tag_of(FUSED_WEIGHT, head, dtype_code(*r.pair)), a + 6, 4);  // (three launches only)
	if(!wt || !on_device(*wt, dev) || wt->scalar_type() != r.pair->scalar_type() || wt->size(0) != C || wt->size(1) != C) return none();
	const Tensor out_weight = *wt, fused = wf ? *wf : Tensor();
	Tensor out;
	int    rc;
	{
		without_gil g;
		if(grid_projected_ok(r, ws)) rc = grid_projected(r, m, ws, turned, hint, exact, out_weight, out, dev);
		else {
			Tensor normed, bias, gated;
			rc = ln_pair_bias(r, normed, bias, dev);
			if(rc == AF3_OK) {
				const Tensor rows = turned ? normed.transpose(0, 1) : normed;
				rc = B * head >= least && !exact ? grid_kernel(rows, m, &bias, ws, head, gated, dev) : 1;
				if(rc == 1 && fused.defined()) {
					const Tensor y = at::linear(rows.reshape({B * N, C}), fused);
					if(y.scalar_type() == normed.scalar_type() && y.is_contiguous()) {
						gated = new_tensor({B, N, C}, y.scalar_type(), dev);
						rc    = attend(y, B, N, head, m, &bias, gated, hint, exact, dev);
					}
				}
			}
			if(rc == AF3_OK) rc = narrow_linear(gated, out_weight, out, dev);
		}
		if(turned && rc == AF3_OK) out = out.transpose(0, 1);
	}
	return rc == 1 ? none() : answer(rc, std::move(out));
	END_HANDLE_TH_ERRORS
}

// ---- gated linear unit --------------------------------------------------------------------------------------------------
// gated_linear_unit(x [.., K], weight [K, 2N], tag of its transposed form)
PyObject* py_gated_linear_unit(PyObject*, PyObject* const* a, Py_ssize_t n) {
	HANDLE_TH_ERRORS
	if(n != 3) return none();
	const Tensor *x = tensor_of(a[0]), *wt = derived_of(PyLong_AsLongLong(a[2]), a + 1, 1);
	const int     dev = device_of(x);
	if(dev < 0 || !wt || x->dim() < 1 || x->numel() == 0 || x->scalar_type() != at::kBFloat16 || wt->scalar_type() != at::kBFloat16 || !on_device(*wt, dev) || !x->is_contiguous() ||
	   reinterpret_cast<uintptr_t>(x->const_data_ptr()) % 16 || x->size(-1) != wt->size(1))
		return none();
	const Tensor weight = *wt;
	Tensor       out;
	int          rc;
	{
		without_gil g;
		const int64_t K = weight.size(1), N = weight.size(0) / 2;
		auto sizes = x->sizes().vec();
		sizes.back() = N;
		out = new_tensor(sizes, at::kBFloat16, dev);
		rc  = af3_gated_linear_unit(x->const_data_ptr(), weight.const_data_ptr(), out.data_ptr(), x->numel() / K, K, N, AF3_BF16, current_stream(dev));
	}
	return answer(rc, std::move(out));
	END_HANDLE_TH_ERRORS
}

// ---- attention to states of another length, relative position bias ------------------------------------------------------------
// A graph that is captured may not wait for work outside of it, and a backward pass runs each operation on the stream that its forward pass ran on: all that leads to the inputs must
// have been recorded within the same capture.  The gradient of a leaf is accumulated on the stream that was current when the leaf first came into a graph of operations
// that is still alive; that must be the capturing stream itself.  Otherwise the engine makes the streams wait for each other and ends the process.  Looked at while capturing only.
void check_capture(at::ArrayRef<const Tensor*> inputs, int dev) {
	hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
	const c10::hip::HIPStream stream = c10::hip::getCurrentHIPStream((c10::DeviceIndex)dev);
	if(hipStreamIsCapturing(stream.stream(), &status) != hipSuccess || status == hipStreamCaptureStatusNone) return;
	unsigned long long capture = 0;
	if(hipStreamGetCaptureInfo(stream.stream(), &status, &capture) != hipSuccess) return;
	auto within = [&](const c10::Stream& s) {
		if(s.id() == stream.id() || s.id() == 0) return s.id() == stream.id();   // (0, the default stream, is never captured and must not be asked)
		hipStreamCaptureStatus of = hipStreamCaptureStatusNone;
		unsigned long long     id = 0;
		return hipStreamGetCaptureInfo(c10::hip::HIPStream(c10::hip::HIPStream::UNCHECKED, s).stream(), &of, &id) == hipSuccess && of == hipStreamCaptureStatusActive && id == capture;
	};
	std::vector<torch::autograd::Node*>        open;
	std::unordered_set<torch::autograd::Node*> seen;
	std::vector<std::shared_ptr<torch::autograd::Node>> leaves;
	auto look = [&](const std::shared_ptr<torch::autograd::Node>& node) {
		if(node && seen.insert(node.get()).second) open.push_back(node.get());
	};
	for(const Tensor* t : inputs) {
		if(!t || !t->defined() || !t->requires_grad()) continue;
		if(t->grad_fn()) look(t->grad_fn());
		else if(auto leaf = torch::autograd::impl::try_get_grad_accumulator(*t)) leaves.push_back(leaf), look(leaf);
	}
	while(!open.empty()) {
		torch::autograd::Node* node = open.back();
		open.pop_back();
		if(const auto own = node->stream()) {
			if(dynamic_cast<torch::autograd::AccumulateGrad*>(node)) {
				TORCH_CHECK(own->id() == stream.id(),
							"a gradient is captured into a HIP graph while a graph of operations recorded on another stream still holds one of its leaves (an earlier result that was not "
							"freed, for instance): the capture would wait for that stream. Free it first, or capture with leaves of their own");
			} else {
				TORCH_CHECK(within(*own), "a gradient is captured into a HIP graph of an input that comes from operations outside of the capture (", node->name(),
							"): the capture would wait for their stream. Detach it, or capture them too");
			}
		}
		for(const auto& e : node->next_edges()) look(e.function);
	}
}
// The gradients as results that know no derivative of their own: asking for one raises.
torch::autograd::variable_list once(torch::autograd::variable_list grads, const char* what) {
	if(!at::GradMode::is_enabled()) return grads;
	torch::autograd::variable_list in;
	for(Tensor& g : grads) in.push_back(g.defined() ? g.detach().requires_grad_(true) : g);
	auto error = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " has no second derivative", (int64_t)in.size());
	return error->apply(std::move(in));
}
// Forward-mode differentiation would come out without a tangent: inputs that have one go to the Python side, which refuses them, and gradients that have one are refused.
bool has_tangent(std::initializer_list<const Tensor*> tensors) {
	for(const Tensor* t : tensors)
		if(t && t->defined() && t->_fw_grad(0).defined()) return true;
	return false;
}
void no_tangent(const Tensor& grad, const char* what) { TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent({&grad}), what, " has no forward-mode derivative"); }
void raise(int rc, const char* what) { TORCH_CHECK(rc == AF3_OK, what, ": ", af3_status_string(rc), " (af3_status ", rc, ")"); }

struct position_call {
	Tensor  table, q_positions, k_positions;
	int64_t Lq, Lk, scheme, both, distance, offset;
	af3_position_bias_params block(at::IntArrayRef table_sizes, at::IntArrayRef strides, at::ScalarType type) const {
		af3_position_bias_params p{};
		if(q_positions.defined()) p.q_positions = static_cast<const int64_t*>(q_positions.const_data_ptr());
		if(k_positions.defined()) p.k_positions = static_cast<const int64_t*>(k_positions.const_data_ptr());
		p.q_offset = offset, p.buckets = table_sizes[0], p.H = table_sizes[1], p.Lq = Lq, p.Lk = Lk, p.max_distance = distance;
		p.table_stride[0] = strides[0], p.table_stride[1] = strides[1];
		p.scheme = (int32_t)scheme, p.bidirectional = (int32_t)both, p.dtype = type == at::kBFloat16 ? AF3_BF16 : AF3_F32;
		return p;
	}
	int forward(Tensor& out) const {
		const int dev = (int)table.get_device();
		af3_position_bias_params p = block(table.sizes(), table.strides(), table.scalar_type());
		out = new_tensor({p.H, Lq, Lk}, table.scalar_type(), dev);
		p.table = table.const_data_ptr(), p.out = out.data_ptr();
		return af3_position_bias_forward(&p, current_stream(dev));
	}
};
// What a bfloat16 gradient of a bias lost by its rounding, on its way from the one attention call that has the bias to the bias's node: that call leaves it here
// in a backward pass, and the node takes it if the gradient that arrives is the very tensor the call made (a bias that something else has too, or whose gradient a
// hook may have changed, has its table's gradient from the gradient that arrives alone).
struct handed_on : torch::CustomClassHolder {
	struct share {
		Tensor  grad, lost;
		int64_t version;
	};
	static constexpr size_t MOST = 8;   // passes through one graph at a time; what a pass that failed left behind goes with newer ones
	Tensor               table;         // an alias of its values: tells whether they were changed in place
	int64_t              version;
	std::atomic<int64_t> calls{0};      // attention calls that have the bias
	std::mutex           lock;
	std::map<int, share> passes;        // by the pass they belong to
	void put(int pass, share s) {
		const std::lock_guard<std::mutex> hold(lock);
		passes[pass] = std::move(s);
		if(passes.size() > MOST) passes.erase(passes.begin());
	}
	Tensor take(int pass, const Tensor& grad) {
		const std::lock_guard<std::mutex> hold(lock);
		const auto it = passes.find(pass);
		if(it == passes.end()) return Tensor();
		const share s = std::move(it->second);
		passes.erase(it);
		return s.grad.is_same(grad) && (int64_t)grad._version() == s.version ? s.lost : Tensor();
	}
};
struct position_function : torch::autograd::Function<position_function> {
	static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& table, const std::optional<Tensor>& given_q, const std::optional<Tensor>& given_k,
					  std::vector<int64_t> s) {
		const Tensor q_positions = given_q.value_or(Tensor()), k_positions = given_k.value_or(Tensor());
		Tensor       out;
		raise(position_call{table, q_positions, k_positions, s[0], s[1], s[2], s[3], s[4], s[5]}.forward(out), "af3_position_bias_forward");
		ctx->save_for_backward({q_positions, k_positions});
		auto handed     = c10::make_intrusive<handed_on>();
		handed->table   = table.detach();
		handed->version = (int64_t)table._version();
		ctx->saved_data["handed"] = at::IValue::make_capsule(std::move(handed));
		s.push_back(table.size(0)), s.push_back(table.size(1));
		ctx->saved_data["settings"] = std::move(s);
		return out;
	}
	static c10::intrusive_ptr<handed_on> handed(torch::autograd::AutogradContext& ctx) { return c10::static_intrusive_pointer_cast<handed_on>(ctx.saved_data["handed"].toCapsule()); }
	// the node that made a tensor, if it is one of these
	static torch::autograd::CppNode<position_function>* node(const std::shared_ptr<torch::autograd::Node>& of) { return dynamic_cast<torch::autograd::CppNode<position_function>*>(of.get()); }
	// the table's gradient [buckets, H] of a gradient g of the bias; with what g's rounding lost (laid out like g): what that misses
	static Tensor sums(Tensor g, const Tensor& lost, const Tensor& q_positions, const Tensor& k_positions, const std::vector<int64_t>& s) {
		const int dev = (int)g.get_device();
		if(!inner_1(g)) g = g.contiguous();
		Tensor out = new_tensor({s[6], s[7]}, g.scalar_type(), dev);
		const position_call call{Tensor(), q_positions, k_positions, s[0], s[1], s[2], s[3], s[4], s[5]};
		af3_position_bias_params p = call.block(out.sizes(), out.strides(), g.scalar_type());
		if(lost.defined()) p.grad_residual = lost.const_data_ptr();
		p.grad = g.const_data_ptr(), p.grad_stride[0] = g.stride(0), p.grad_stride[1] = g.stride(1), p.out = out.data_ptr();
		const int64_t bytes = af3_position_bias_workspace_bytes(&p);
		raise(bytes < 0 ? (int)bytes : AF3_OK, "af3_position_bias_workspace_bytes");
		const at::DataPtr ws = new_scratch(bytes);
		p.workspace = ws.get(), p.workspace_bytes = bytes;
		raise(af3_position_bias_backward(&p, current_stream(dev)), "af3_position_bias_backward");
		return out;
	}
	static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grad_out) {
		torch::autograd::variable_list grads(4);
		no_tangent(grad_out[0], "the gradient of relative_position_bias");
		{
			at::AutoGradMode none(false);
			const auto   saved = ctx->get_saved_variables();
			const auto   settings = ctx->saved_data["settings"].toIntVector();
			const Tensor lost = handed(*ctx)->take(torch::autograd::get_current_graph_task_id(), grad_out[0]);
			grads[0] = sums(grad_out[0], Tensor(), saved[0], saved[1], settings);
			if(lost.defined()) {
				// (lost belongs to the attention call's stream, which need not be this one)
				c10::hip::HIPCachingAllocator::recordStream(lost.storage().data_ptr(), c10::hip::getCurrentHIPStream((c10::DeviceIndex)lost.get_device()));
				grads[0].add_(sums(grad_out[0], lost, saved[0], saved[1], settings));
			}
		}
		return once(std::move(grads), "relative_position_bias");
	}
};

struct cross_call {
	Tensor         q, k, v, mask, bias;   // mask as bytes [1|B, Lk] or undefined, bias undefined: none
	double         scale;
	af3_cross_attention_params block() const {
		af3_cross_attention_params p{};
		p.q = q.const_data_ptr(), p.k = k.const_data_ptr(), p.v = v.const_data_ptr();
		p.B = q.size(0), p.H = q.size(1), p.Lq = q.size(2), p.D = q.size(3), p.Hkv = k.size(1), p.Lk = k.size(2);
		put_strides(p.q_stride, q), put_strides(p.k_stride, k), put_strides(p.v_stride, v);
		if(bias.defined()) p.bias = bias.const_data_ptr(), p.bias_stride[0] = bias.stride(0), p.bias_stride[1] = bias.stride(1);
		if(mask.defined()) p.key_mask = static_cast<const uint8_t*>(mask.const_data_ptr()), p.key_mask_stride_b = mask.dim() > 1 && mask.size(0) != 1 ? mask.stride(0) : 0;
		p.dtype = dtype_code(q), p.softmax_scale = (float)scale;
		return p;
	}
	int forward(Tensor& out, Tensor* stats, Tensor* lost) const {
		const int dev = (int)q.get_device();
		out = new_tensor(q.sizes(), q.scalar_type(), dev);
		af3_cross_attention_params p = block();
		p.out = out.data_ptr();
		put_strides(p.out_stride, out);
		if(stats) {
			*stats  = new_tensor({p.B, p.H, p.Lq, 2}, at::kFloat, dev);
			p.stats = static_cast<float*>(stats->data_ptr());
			if(p.dtype == AF3_BF16) *lost = new_tensor(q.sizes(), q.scalar_type(), dev), p.out_residual = lost->data_ptr();
		}
		at::DataPtr   ws;
		const int64_t bytes = af3_cross_attention_workspace_bytes(&p);
		if(bytes < 0) return (int)bytes;
		if(bytes > 0) ws = new_scratch(bytes), p.workspace = ws.get(), p.workspace_bytes = bytes;
		return af3_cross_attention_forward(&p, current_stream(dev));
	}
};
// The gradient of a bfloat16 bias is rounded to bfloat16, as that of a bfloat16 tensor has to be.  Where the bias came straight out of relative_position_bias and nothing
// else has it, what the rounding lost is handed on to its node, and the table's gradient is rounded once.
struct cross_function : torch::autograd::Function<cross_function> {
	static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const std::optional<Tensor>& given_bias,
					  const std::optional<Tensor>& given_mask, double scale, bool hands_on) {
		const Tensor bias = given_bias.value_or(Tensor()), mask = given_mask.value_or(Tensor());
		Tensor       out, stats, lost;
		raise(cross_call{q, k, v, mask, bias, scale}.forward(out, &stats, &lost), "af3_cross_attention_forward");
		ctx->save_for_backward({q, k, v, bias, mask, out, stats, lost});
		ctx->saved_data["scale"] = scale, ctx->saved_data["hands_on"] = hands_on;
		return out;
	}
	// where what the bias's gradient loses goes in this pass: to the bias's node, if that will run and nobody gets to see the gradient on its way
	static c10::intrusive_ptr<handed_on> receiver(bool hands_on) {
		if(!hands_on || at::GradMode::is_enabled()) return {};   // (a graph of the gradient is wanted: it must hold for the gradient as it stands)
		const auto self = torch::autograd::get_current_node();
		auto* const to  = self ? position_function::node(self->next_edge(3).function) : nullptr;
		if(!to || !self->post_hooks().empty() || !to->pre_hooks().empty() || !to->tensor_pre_hooks().empty()) return {};
		if(const auto* const info = torch::autograd::get_current_graph_task_exec_info(); info && !info->empty()) {
			const auto it = info->find(to);
			if(it == info->end() || !it->second.needed_) return {};
		}
		const auto handed = position_function::handed(to->ctx_);
		return handed->calls == 1 ? handed : c10::intrusive_ptr<handed_on>();
	}
	static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grad_out) {
		const auto saved = ctx->get_saved_variables();
		const cross_call call{saved[0], saved[1], saved[2], saved[4], saved[3], ctx->saved_data["scale"].toDouble()};
		const int        dev = (int)call.q.get_device();
		Tensor           g = grad_out[0];
		no_tangent(g, "the gradient of cross_attention");
		torch::autograd::variable_list grads(7);
		Tensor           bias_lost;
		const auto       handed = receiver(ctx->saved_data["hands_on"].toBool());
		{
			at::AutoGradMode none(false);
			if(!inner_1(g)) g = g.contiguous();
			af3_cross_attention_params p = call.block();
			p.out = saved[5].data_ptr(), p.stats = static_cast<float*>(saved[6].data_ptr());
			put_strides(p.out_stride, saved[5]);
			if(saved[7].defined()) p.out_residual = saved[7].data_ptr();
			af3_cross_attention_grads o{};
			o.grad_out = g.const_data_ptr();
			put_strides(o.grad_out_stride, g);
			auto want = [&](int i, at::IntArrayRef sizes) -> void* {
				if(!ctx->needs_input_grad((size_t)i)) return nullptr;
				grads[i] = new_tensor(sizes, call.q.scalar_type(), dev);
				return grads[i].data_ptr();
			};
			o.grad_q = want(0, call.q.sizes()), o.grad_k = want(1, call.k.sizes()), o.grad_v = want(2, call.v.sizes());
			if(call.bias.defined()) o.grad_bias = want(3, call.bias.sizes());
			if(o.grad_bias && handed) bias_lost = new_tensor(call.bias.sizes(), call.q.scalar_type(), dev), o.grad_bias_residual = bias_lost.data_ptr();
			const int64_t     bytes = af3_cross_attention_backward_workspace_bytes(&p);
			raise(bytes < 0 ? (int)bytes : AF3_OK, "af3_cross_attention_backward_workspace_bytes");
			const at::DataPtr ws = new_scratch(bytes);
			o.workspace = ws.get(), o.workspace_bytes = bytes;
			raise(af3_cross_attention_backward(&p, &o, current_stream(dev)), "af3_cross_attention_backward");
			if(bias_lost.defined()) handed->put(torch::autograd::get_current_graph_task_id(), {grads[3], bias_lost, (int64_t)grads[3]._version()});
		}
		return once(std::move(grads), "cross_attention");
	}
};
std::optional<Tensor> given(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }
bool wants_grad(std::initializer_list<const Tensor*> tensors) {
	if(!at::GradMode::is_enabled()) return false;
	for(const Tensor* t : tensors)
		if(t && t->defined() && t->requires_grad()) return true;
	return false;
}
Tensor apply_cross(const cross_call& c) {
	bool hands_on = false;
	if(c.bias.defined() && c.bias.scalar_type() == at::kBFloat16 && c.bias.requires_grad() && c.q.size(1) <= 0x7fff)   // (heads: as many as the sums take with a residual)
		if(auto* const node = position_function::node(c.bias.grad_fn())) {
			const auto handed = position_function::handed(node->ctx_);
			handed->calls++;
			hands_on = (int64_t)handed->table._version() == handed->version;   // (a table changed in place since: the bias's gradient alone)
		}
	return cross_function::apply(c.q, c.k, c.v, given(c.bias), given(c.mask), c.scale, hands_on);
}
// cross_attention(q, k, v, mask, bias, scale or None)
PyObject* py_cross_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
	HANDLE_TH_ERRORS
	if(n != 6) return none();
	const Tensor *q = tensor_of(a[0]), *k = tensor_of(a[1]), *v = tensor_of(a[2]);
	if(!q || !k || !v || q->dim() != 4 || k->dim() != 4 || k->sizes() != v->sizes() || q->numel() == 0 || k->numel() == 0) return none();
	const int dev = device_of(q);
	const auto type = q->scalar_type();
	if(dev < 0 || dtype_code(*q) < 0 || k->scalar_type() != type || v->scalar_type() != type || !on_device(*k, dev) || !on_device(*v, dev) || !inner_1(*q) || !inner_1(*k) || !inner_1(*v)) return none();
	const int64_t B = q->size(0), H = q->size(1), Lq = q->size(2), D = q->size(3), Lk = k->size(2);
	if(k->size(0) != B || k->size(3) != D || H % k->size(1) != 0 || D > AF3_DPA_MAX_HEAD_DIM) return none();
	cross_call c{*q, *k, *v, Tensor(), Tensor(), 0.0};
	key_mask   m;
	if(!mask_of(a[3], B, Lk, dev, m)) return none();
	if(a[3] != Py_None) {
		const Tensor& t = *tensor_of(a[3]);
		c.mask = t.dim() == 4 ? t.as_strided({t.size(0), Lk}, {t.stride(0), 1}) : t;
	}
	if(a[4] != Py_None) {
		const Tensor* t = tensor_of(a[4]);
		if(!t || !on_device(*t, dev) || t->scalar_type() != type || t->dim() != 3 || t->size(0) != H || t->size(1) != Lq || t->size(2) != Lk || !inner_1(*t)) return none();
		c.bias = *t;
	}
	c.scale = a[5] == Py_None ? std::pow((double)D, -0.5) : PyFloat_AsDouble(a[5]);
	if(PyErr_Occurred()) {
		PyErr_Clear();
		return none();
	}
	if(!(c.scale > 0.0 && (float)c.scale > 0.f && (float)c.scale < INFINITY) || has_tangent({q, k, v, &c.bias})) return none();
	Tensor out;
	int    rc = AF3_OK;
	const bool graph = wants_grad({q, k, v, &c.bias});
	// (sizes whose gradients would be refused: the Python side says so)
	if(graph && (B * k->size(1) * ((Lk + 31) / 32) > 0xffffff || (c.bias.defined() && c.bias.requires_grad() && H * ((Lq + 63) / 64) * ((Lk + 63) / 64) > 0xffffff))) return none();
	{
		without_gil g;
		if(graph) check_capture({q, k, v, &c.bias}, dev), out = apply_cross(c);
		else rc = c.forward(out, nullptr, nullptr);
	}
	return answer(rc, std::move(out));
	END_HANDLE_TH_ERRORS
}

bool positions_of(PyObject* o, int64_t n, int dev, Tensor& t) {
	if(o == Py_None) return true;
	const Tensor* x = tensor_of(o);
	if(!x || !on_device(*x, dev) || x->scalar_type() != at::kLong || x->dim() != 1 || x->size(0) != n || !x->is_contiguous()) return false;
	t = *x;
	return true;
}
// position_bias(table, q_len, k_len, scheme, bidirectional, max_distance, q_positions, k_positions, q_offset); scheme as its number
PyObject* py_position_bias(PyObject*, PyObject* const* a, Py_ssize_t n) {
	HANDLE_TH_ERRORS
	if(n != 9) return none();
	const Tensor* table = tensor_of(a[0]);
	const int     dev   = device_of(table);
	if(dev < 0 || table->dim() != 2 || dtype_code(*table) < 0 || table->numel() == 0 || has_tangent({table})) return none();
	int64_t number[5];   // q_len, k_len, scheme, max_distance, q_offset
	const int at[5] = {1, 2, 3, 5, 8};
	for(int i = 0; i < 5; i++) {
		if(!PyLong_CheckExact(a[at[i]])) return none();
		number[i] = PyLong_AsLongLong(a[at[i]]);
	}
	if(PyErr_Occurred()) {
		PyErr_Clear();
		return none();
	}
	position_call c{*table, Tensor(), Tensor(), number[0], number[1], number[2], a[4] == Py_True, number[3], number[4]};
	if((a[4] != Py_True && a[4] != Py_False) || c.Lq < 1 || c.Lk < 1 || !positions_of(a[6], c.Lq, dev, c.q_positions) || !positions_of(a[7], c.Lk, dev, c.k_positions)) return none();
	const af3_position_bias_params p = c.block(table->sizes(), table->strides(), table->scalar_type());
	if(af3_position_bias_workspace_bytes(&p) < 0) return none();   // (settings that do not go together: the Python side says what is wrong)
	Tensor     out;
	int        rc = AF3_OK;
	const bool graph = wants_grad({table});
	{
		without_gil g;
		if(graph) check_capture({table}, dev), out = position_function::apply(c.table, given(c.q_positions), given(c.k_positions), std::vector<int64_t>{c.Lq, c.Lk, c.scheme, c.both, c.distance, c.offset});
		else rc = c.forward(out);
	}
	return answer(rc, std::move(out));
	END_HANDLE_TH_ERRORS
}
// ---- rotary positions ------------------------------------------------------------------------------------------------------------
PyObject* pair(Tensor&& a, Tensor&& b) {   // (an undefined tensor: None)
	PyObject* const x = a.defined() ? wrap(std::move(a)) : Py_NewRef(Py_None);
	PyObject* const y = b.defined() ? wrap(std::move(b)) : Py_NewRef(Py_None);
	PyObject* const t = PyTuple_New(2);
	PyTuple_SET_ITEM(t, 0, x), PyTuple_SET_ITEM(t, 1, y);
	return t;
}
struct rotary_call {
	Tensor  frequencies, positions;   // positions [L] or [1|B, L] or undefined
	int64_t offset;
	bool    interleaved;
	double  scale;
	// x[i] [B, heads, L, D], undefined: none; out[i] likewise
	int run(const Tensor (&x)[2], Tensor (&out)[2], bool inverse) const {
		af3_rotary_params p{};
		int               n = 0, dev = 0;
		for(int i = 0; i < 2; i++) {
			if(!x[i].defined()) continue;
			dev    = (int)x[i].get_device();
			out[i] = new_tensor(x[i].sizes(), x[i].scalar_type(), dev);
			p.x[n] = x[i].const_data_ptr(), p.out[n] = out[i].data_ptr(), p.heads[n] = x[i].size(1);
			put_strides(p.x_stride[n], x[i]), put_strides(p.out_stride[n], out[i]);
			p.B = x[i].size(0), p.L = x[i].size(2), p.D = x[i].size(3), p.dtype = dtype_code(x[i]);
			n++;
		}
		p.frequencies = frequencies.const_data_ptr<double>(), p.rotary = 2 * frequencies.size(0);
		if(positions.defined()) p.positions = positions.const_data_ptr<int64_t>(), p.position_stride_b = positions.dim() > 1 && positions.size(0) != 1 ? positions.stride(0) : 0;
		p.offset = offset, p.interleaved = interleaved, p.inverse = inverse, p.scale = (float)scale;
		return af3_rotary_embedding(&p, current_stream(dev));
	}
};
struct rotary_function : torch::autograd::Function<rotary_function> {
	static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const std::optional<Tensor>& k, const Tensor& frequencies,
												  const std::optional<Tensor>& positions, int64_t offset, bool interleaved, double scale) {
		const Tensor x[2] = {q, k.value_or(Tensor())};
		Tensor       out[2];
		raise(rotary_call{frequencies, positions.value_or(Tensor()), offset, interleaved, scale}.run(x, out, false), "af3_rotary_embedding");
		ctx->save_for_backward({frequencies, positions.value_or(Tensor())});
		ctx->saved_data["offset"] = offset, ctx->saved_data["interleaved"] = interleaved, ctx->saved_data["scale"] = scale;
		ctx->set_materialize_grads(false);
		if(!out[1].defined()) return {out[0]};
		return {out[0], out[1]};
	}
	static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grad_out) {
		torch::autograd::variable_list grads(7);
		for(const Tensor& g : grad_out) no_tangent(g, "the gradient of rotary_embedding");
		{
			at::AutoGradMode none(false);
			const auto       saved = ctx->get_saved_variables();
			Tensor           g[2], out[2];
			for(size_t i = 0; i < grad_out.size(); i++)
				if(grad_out[i].defined() && ctx->needs_input_grad(i)) g[i] = inner_1(grad_out[i]) ? grad_out[i] : grad_out[i].contiguous();
			if(g[0].defined() || g[1].defined())
				raise(rotary_call{saved[0], saved[1], ctx->saved_data["offset"].toInt(), ctx->saved_data["interleaved"].toBool(), ctx->saved_data["scale"].toDouble()}.run(g, out, true), "af3_rotary_embedding");
			grads[0] = out[0], grads[1] = out[1];
		}
		return once(std::move(grads), "rotary_embedding");
	}
};
bool number_of(PyObject* o, int64_t& n) {
	if(!PyLong_CheckExact(o)) return false;
	n = PyLong_AsLongLong(o);
	if(!PyErr_Occurred()) return true;
	PyErr_Clear();
	return false;
}
bool real_of(PyObject* o, double& x) {
	if(!PyFloat_CheckExact(o)) return false;
	x = PyFloat_AS_DOUBLE(o);
	return true;
}
bool truth_of(PyObject* o, bool& x) {
	x = o == Py_True;
	return o == Py_True || o == Py_False;
}
// rotary(q, k or None, frequencies, positions or None, offset, interleaved, scale): (q, k or None) turned
PyObject* py_rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
	HANDLE_TH_ERRORS
	if(n != 7) return none();
	const Tensor *q = tensor_of(a[0]), *k = a[1] == Py_None ? nullptr : tensor_of(a[1]), *f = tensor_of(a[2]);
	const int     dev = device_of(q);
	if(dev < 0 || (!k && a[1] != Py_None) || !f || q->dim() != 4 || q->numel() == 0 || dtype_code(*q) < 0 || !inner_1(*q)) return none();
	if(k && (!on_device(*k, dev) || k->dim() != 4 || k->scalar_type() != q->scalar_type() || k->size(0) != q->size(0) || k->size(2) != q->size(2) || k->size(3) != q->size(3) || k->numel() == 0 || !inner_1(*k)))
		return none();
	if(!on_device(*f, dev) || f->dim() != 1 || f->scalar_type() != at::kDouble || !f->is_contiguous() || f->requires_grad() || f->size(0) < 1 || 2 * f->size(0) > q->size(3) || q->size(3) > AF3_ROTARY_MAX_HEAD_DIM) return none();
	rotary_call c{*f, Tensor(), 0, false, 1.0};
	if(a[3] != Py_None) {
		const Tensor* t = tensor_of(a[3]);
		if(!t || !on_device(*t, dev) || t->scalar_type() != at::kLong || (t->dim() != 1 && t->dim() != 2) || t->size(-1) != q->size(2) || !inner_1(*t) || (t->dim() == 2 && t->size(0) != 1 && t->size(0) != q->size(0))) return none();
		c.positions = *t;
	}
	if(!number_of(a[4], c.offset) || !truth_of(a[5], c.interleaved) || !real_of(a[6], c.scale) || !std::isfinite((float)c.scale) || c.offset > ((int64_t)1 << 62) || c.offset < -((int64_t)1 << 62) || has_tangent({q, k, f})) return none();
	const Tensor x[2] = {*q, k ? *k : Tensor()};
	Tensor       out[2];
	int          rc = AF3_OK;
	{
		without_gil g;
		if(wants_grad({q, k})) {
			check_capture({q, k}, dev);
			auto r = rotary_function::apply(x[0], given(x[1]), c.frequencies, given(c.positions), c.offset, c.interleaved, c.scale);
			out[0] = r[0];
			if(r.size() > 1) out[1] = r[1];
		} else rc = c.run(x, out, false);
	}
	return rc == AF3_OK ? pair(std::move(out[0]), std::move(out[1])) : PyLong_FromLong(rc);
	END_HANDLE_TH_ERRORS
}

// ---- norms around a block ----------------------------------------------------------------------------------------------------------
// the distance of a tensor's rows [.., C] where they are equally far apart, -1 otherwise
int64_t row_stride(const Tensor& t) {
	int64_t stride = -1, behind = 1;   // of the axes seen so far, from the last; rows behind this axis
	for(int64_t i = t.dim() - 2; i >= 0; i--) {
		if(t.size(i) == 1) continue;
		if(stride < 0) stride = t.stride(i);
		else if(t.stride(i) != stride * behind) return -1;
		behind *= t.size(i);
	}
	return stride < 0 ? t.size(-1) : stride;
}
struct norm_call {
	Tensor  x, y, gate, weight, bias, post_weight;
	int64_t norm, post_norm, sigmoid;
	double  scale, eps;
	// how a parameter's rows go with those of y; -1: not as the kernels take them
	static int share(const Tensor& t, const Tensor& y, int64_t& group) {
		if(!t.defined()) return AF3_SHARE_NONE;
		const int64_t C = y.size(-1), rows = y.numel() / C;
		if(!t.is_contiguous() || t.size(-1) != C) return -1;
		if(t.numel() == C) return t.dim() == 1 || t.dim() == y.dim() ? AF3_SHARE_CHANNEL : -1;
		if(t.dim() != y.dim()) return -1;
		int64_t i = 0, each = 1;
		while(i < y.dim() - 1 && t.size(i) == y.size(i)) i++;
		for(; i < y.dim() - 1; i++) {
			if(t.size(i) != 1) return -1;
			each *= y.size(i);
		}
		if(each == 1) return AF3_SHARE_ROW;
		if(each == rows) return AF3_SHARE_CHANNEL;
		if(group != 0 && group != each) return -1;
		group = each;
		return AF3_SHARE_GROUP;
	}
	bool block(af3_residual_norm_params& p) const {
		p   = af3_residual_norm_params{};
		p.C = y.size(-1), p.rows = y.numel() / p.C;
		p.y = y.const_data_ptr(), p.y_stride = row_stride(y);
		if(x.defined()) p.x = x.const_data_ptr(), p.x_stride = row_stride(x);
		const Tensor* const of[3] = {&gate, &weight, &bias};
		const void**        to[3] = {&p.gate, &p.weight, &p.bias};
		int32_t*            shares[3] = {&p.gate_share, &p.weight_share, &p.bias_share};
		for(int i = 0; i < 3; i++) {
			if((*shares[i] = share(*of[i], y, p.group)) < 0) return false;
			if(of[i]->defined()) *to[i] = of[i]->const_data_ptr();
		}
		if(post_weight.defined()) {
			if(post_weight.dim() != 1 || post_weight.size(0) != p.C || !post_weight.is_contiguous()) return false;
			p.post_weight = post_weight.const_data_ptr();
		}
		p.norm = (int32_t)norm, p.post_norm = (int32_t)post_norm, p.gate_sigmoid = (int32_t)sigmoid, p.dtype = dtype_code(y);
		p.eps = (float)eps, p.residual_scale = (float)scale;
		return p.y_stride >= 0 && p.x_stride >= 0;
	}
	int forward(Tensor& out, Tensor& normed, Tensor* stats) const {
		const int                dev = (int)y.get_device();
		af3_residual_norm_params p;
		if(!block(p)) return AF3_ERR_BAD_ARGUMENT;
		out = new_tensor(y.sizes(), y.scalar_type(), dev), p.out = out.data_ptr();
		if(norm != AF3_NORM_NONE) normed = new_tensor(y.sizes(), y.scalar_type(), dev), p.normed = normed.data_ptr();
		if(stats) *stats = new_tensor({p.rows, 4}, at::kFloat, dev), p.stats = static_cast<float*>(stats->data_ptr());
		return af3_residual_norm_forward(&p, current_stream(dev));
	}
};
struct norm_function : torch::autograd::Function<norm_function> {
	static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const std::optional<Tensor>& x, const Tensor& y, const std::optional<Tensor>& weight,
												  const std::optional<Tensor>& bias, const std::optional<Tensor>& gate, const std::optional<Tensor>& post_weight, std::vector<int64_t> kinds,
												  double scale, double eps) {
		const norm_call c{x.value_or(Tensor()), y, gate.value_or(Tensor()), weight.value_or(Tensor()), bias.value_or(Tensor()), post_weight.value_or(Tensor()), kinds[0], kinds[1], kinds[2], scale, eps};
		Tensor          out, normed, stats;
		raise(c.forward(out, normed, &stats), "af3_residual_norm_forward");
		ctx->save_for_backward({c.x, y, c.weight, c.bias, c.gate, c.post_weight, stats});
		ctx->saved_data["kinds"] = std::move(kinds), ctx->saved_data["scale"] = scale, ctx->saved_data["eps"] = eps;
		ctx->set_materialize_grads(false);
		if(!normed.defined()) return {out};
		return {out, normed};
	}
	static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grad_out) {
		torch::autograd::variable_list grads(9);
		for(const Tensor& g : grad_out) no_tangent(g, "the gradient of residual_norm");
		{
			at::AutoGradMode none(false);
			const auto       saved = ctx->get_saved_variables();
			const auto       kinds = ctx->saved_data["kinds"].toIntVector();
			const norm_call  c{saved[0], saved[1], saved[4], saved[2], saved[3], saved[5], kinds[0], kinds[1], kinds[2], ctx->saved_data["scale"].toDouble(), ctx->saved_data["eps"].toDouble()};
			const int        dev = (int)c.y.get_device();
			af3_residual_norm_params p;
			af3_residual_norm_grads  o{};
			raise(c.block(p) ? AF3_OK : AF3_ERR_BAD_ARGUMENT, "af3_residual_norm_backward");
			p.stats = static_cast<float*>(saved[6].data_ptr());
			Tensor g[2];
			for(size_t i = 0; i < grad_out.size(); i++)
				if(grad_out[i].defined()) g[i] = inner_1(grad_out[i]) && row_stride(grad_out[i]) >= 0 ? grad_out[i] : grad_out[i].contiguous();
			if(g[0].defined()) o.grad_out = g[0].const_data_ptr(), o.grad_out_stride = row_stride(g[0]);
			if(g[1].defined()) o.grad_normed = g[1].const_data_ptr(), o.grad_normed_stride = row_stride(g[1]);
			const bool reached = g[0].defined() || g[1].defined();   // (a consumer of both results may have no gradient for either)
			bool   any  = false;
			size_t edge = 0;   // (tensors that were not given have none)
			auto want = [&](int i, const Tensor& like, bool from) -> void* {   // `from`: a gradient comes from where this one is made of
				if(!like.defined() || !ctx->needs_input_grad(edge++)) return nullptr;
				grads[i] = new_tensor(like.sizes(), like.scalar_type(), dev);
				if(!from) {
					grads[i].zero_();
					return nullptr;
				}
				any = true;
				return grads[i].data_ptr();
			};
			o.grad_x = want(0, c.x, reached), o.grad_y = want(1, c.y, reached), o.grad_weight = want(2, c.weight, g[1].defined()), o.grad_bias = want(3, c.bias, g[1].defined());
			o.grad_gate = want(4, c.gate, reached), o.grad_post_weight = want(5, c.post_weight, reached);
			if(any) {
				const int64_t bytes = af3_residual_norm_backward_workspace_bytes(&p, &o);
				raise(bytes < 0 ? (int)bytes : AF3_OK, "af3_residual_norm_backward_workspace_bytes");
				at::DataPtr ws;
				if(bytes > 0) ws = new_scratch(bytes), o.workspace = ws.get(), o.workspace_bytes = bytes;
				raise(af3_residual_norm_backward(&p, &o, current_stream(dev)), "af3_residual_norm_backward");
			}
		}
		return once(std::move(grads), "residual_norm");
	}
};
// residual_norm(x or None, y, weight, bias, gate, post_weight, norm, post_norm, sigmoid, residual_scale, eps): (out, normed or None)
PyObject* py_residual_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
	HANDLE_TH_ERRORS
	if(n != 11) return none();
	const Tensor* y   = tensor_of(a[1]);
	const int     dev = device_of(y);
	if(dev < 0 || y->dim() < 1 || y->numel() == 0 || dtype_code(*y) < 0 || !inner_1(*y) || y->size(-1) > AF3_RESIDUAL_NORM_MAX_CHANNELS) return none();
	norm_call c{Tensor(), *y, Tensor(), Tensor(), Tensor(), Tensor(), 0, 0, 0, 1.0, 0.0};
	Tensor*   to[5] = {&c.x, &c.weight, &c.bias, &c.gate, &c.post_weight};
	const int from[5] = {0, 2, 3, 4, 5};
	for(int i = 0; i < 5; i++) {
		if(a[from[i]] == Py_None) continue;
		const Tensor* t = tensor_of(a[from[i]]);
		if(!t || !on_device(*t, dev) || t->scalar_type() != y->scalar_type() || t->dim() < 1 || t->numel() == 0 || !inner_1(*t)) return none();
		*to[i] = *t;
	}
	bool sigmoid;
	if(!number_of(a[6], c.norm) || !number_of(a[7], c.post_norm) || !truth_of(a[8], sigmoid) || !real_of(a[9], c.scale) || !real_of(a[10], c.eps)) return none();
	c.sigmoid = sigmoid;
	if(c.norm < 0 || c.norm > 2 || c.post_norm < 0 || c.post_norm > 2 || (c.norm == 0 && (c.weight.defined() || c.bias.defined())) || (c.post_norm == 0 && c.post_weight.defined()) || (sigmoid && !c.gate.defined())) return none();
	if(!(c.eps >= 0.0) || !std::isfinite((float)c.eps) || !std::isfinite((float)c.scale) || (c.x.defined() && c.x.sizes() != y->sizes()) || has_tangent({&c.x, y, &c.weight, &c.bias, &c.gate, &c.post_weight})) return none();
	af3_residual_norm_params p;
	if(!c.block(p)) return none();   // (parameters or strides that the Python side lays out anew, or refuses)
	Tensor out, normed;
	int    rc = AF3_OK;
	{
		without_gil g;
		const std::initializer_list<const Tensor*> all = {&c.x, &c.y, &c.weight, &c.bias, &c.gate, &c.post_weight};
		if(wants_grad(all)) {
			check_capture(all, dev);
			auto r = norm_function::apply(given(c.x), c.y, given(c.weight), given(c.bias), given(c.gate), given(c.post_weight), std::vector<int64_t>{c.norm, c.post_norm, c.sigmoid}, c.scale, c.eps);
			out = r[0];
			if(r.size() > 1) normed = r[1];
		} else rc = c.forward(out, normed, nullptr);
	}
	return rc == AF3_OK ? pair(std::move(out), std::move(normed)) : PyLong_FromLong(rc);
	END_HANDLE_TH_ERRORS
}

// ---- differential attention --------------------------------------------------------------------------------------------------------
struct diff_call {
	Tensor  q, k, v, lam, mask;   // mask as bytes [1|B, Lk] or undefined
	double  scale;
	int64_t causal, offset;
	af3_diff_attention_params block() const {
		af3_diff_attention_params p{};
		p.q = q.const_data_ptr(), p.k = k.const_data_ptr(), p.v = v.const_data_ptr(), p.lam = lam.const_data_ptr();
		p.B = q.size(0), p.H = q.size(1) / 2, p.Lq = q.size(2), p.D = q.size(3), p.Hkv = v.size(1), p.Lk = k.size(2), p.Dv = v.size(3);
		put_strides(p.q_stride, q), put_strides(p.k_stride, k), put_strides(p.v_stride, v);
		if(mask.defined()) p.key_mask = static_cast<const uint8_t*>(mask.const_data_ptr()), p.key_mask_stride_b = mask.dim() > 1 && mask.size(0) != 1 ? mask.stride(0) : 0;
		p.lam_stride = lam.stride(0), p.lam_dtype = dtype_code(lam), p.dtype = dtype_code(q);
		p.causal = (int32_t)causal, p.q_offset = offset, p.softmax_scale = (float)scale;
		return p;
	}
	int forward(Tensor& out, Tensor* stats, Tensor* second, Tensor* lost) const {
		const int dev = (int)q.get_device();
		af3_diff_attention_params p = block();
		out   = new_tensor({p.B, p.H, p.Lq, p.Dv}, q.scalar_type(), dev);
		p.out = out.data_ptr();
		put_strides(p.out_stride, out);
		if(stats) {
			*stats = new_tensor({p.B, 2 * p.H, p.Lq, 2}, at::kFloat, dev), *second = new_tensor(out.sizes(), q.scalar_type(), dev);
			p.stats = static_cast<float*>(stats->data_ptr()), p.second = second->data_ptr();
			if(p.dtype == AF3_BF16) *lost = new_tensor({2, p.B, p.H, p.Lq, p.Dv}, q.scalar_type(), dev), p.residuals = lost->data_ptr();
		}
		at::DataPtr   ws;
		const int64_t bytes = af3_diff_attention_workspace_bytes(&p);
		if(bytes < 0) return (int)bytes;
		if(bytes > 0) ws = new_scratch(bytes), p.workspace = ws.get(), p.workspace_bytes = bytes;
		return af3_diff_attention_forward(&p, current_stream(dev));
	}
};
struct diff_function : torch::autograd::Function<diff_function> {
	static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lam, const std::optional<Tensor>& given_mask, double scale,
						  int64_t causal, int64_t offset) {
		const Tensor mask = given_mask.value_or(Tensor());
		Tensor       out, stats, second, lost;
		raise(diff_call{q, k, v, lam, mask, scale, causal, offset}.forward(out, &stats, &second, &lost), "af3_diff_attention_forward");
		ctx->save_for_backward({q, k, v, lam, mask, out, stats, second, lost});
		ctx->saved_data["scale"] = scale, ctx->saved_data["causal"] = causal, ctx->saved_data["offset"] = offset;
		return out;
	}
	static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grad_out) {
		const auto      saved = ctx->get_saved_variables();
		const diff_call call{saved[0], saved[1], saved[2], saved[3], saved[4], ctx->saved_data["scale"].toDouble(), ctx->saved_data["causal"].toInt(), ctx->saved_data["offset"].toInt()};
		const int       dev = (int)call.q.get_device();
		Tensor          g = grad_out[0];
		no_tangent(g, "the gradient of differential_attention");
		torch::autograd::variable_list grads(8);
		{
			at::AutoGradMode none(false);
			if(!inner_1(g) || g.stride(2) * (int64_t)g.element_size() >= AF3_DIFF_ATTENTION_GRAD_ROW_BYTES) g = g.contiguous();
			af3_diff_attention_params p = call.block();
			p.out = saved[5].data_ptr(), p.stats = static_cast<float*>(saved[6].data_ptr()), p.second = saved[7].data_ptr();
			if(saved[8].defined()) p.residuals = saved[8].data_ptr();
			put_strides(p.out_stride, saved[5]);
			af3_diff_attention_grads o{};
			o.grad_out = g.const_data_ptr();
			put_strides(o.grad_out_stride, g);
			auto want = [&](int i, const Tensor& like) -> void* {
				if(!ctx->needs_input_grad((size_t)i)) return nullptr;
				grads[i] = new_tensor(like.sizes(), like.scalar_type(), dev);
				return grads[i].data_ptr();
			};
			o.grad_q = want(0, call.q), o.grad_k = want(1, call.k), o.grad_v = want(2, call.v), o.grad_lam = want(3, call.lam);
			const int64_t     bytes = af3_diff_attention_backward_workspace_bytes(&p);
			raise(bytes < 0 ? (int)bytes : AF3_OK, "af3_diff_attention_backward_workspace_bytes");
			const at::DataPtr ws = new_scratch(bytes);
			o.workspace = ws.get(), o.workspace_bytes = bytes;
			raise(af3_diff_attention_backward(&p, &o, current_stream(dev)), "af3_diff_attention_backward");
		}
		return once(std::move(grads), "differential_attention");
	}
};
// differential_attention(q, k, v, lam, mask, causal, q_offset, scale or None)
PyObject* py_differential_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
	HANDLE_TH_ERRORS
	if(n != 8) return none();
	const Tensor *q = tensor_of(a[0]), *k = tensor_of(a[1]), *v = tensor_of(a[2]), *lam = tensor_of(a[3]);
	if(!q || !k || !v || !lam || q->dim() != 4 || k->dim() != 4 || v->dim() != 4 || lam->dim() != 1 || q->numel() == 0 || k->numel() == 0 || v->numel() == 0) return none();
	const int  dev  = device_of(q);
	const auto type = q->scalar_type();
	if(dev < 0 || dtype_code(*q) < 0 || k->scalar_type() != type || v->scalar_type() != type || (lam->scalar_type() != type && lam->scalar_type() != at::kFloat)) return none();
	if(!on_device(*k, dev) || !on_device(*v, dev) || !on_device(*lam, dev) || !inner_1(*q) || !inner_1(*k) || !inner_1(*v)) return none();
	const int64_t B = q->size(0), H = q->size(1) / 2, Hkv = v->size(1), Lk = k->size(2), D = q->size(3), most = type == at::kFloat ? 64 : 128;
	if(q->size(1) != 2 * H || k->size(1) != 2 * Hkv || H % Hkv != 0 || lam->size(0) != H || k->size(0) != B || v->size(0) != B || k->size(3) != D || v->size(2) != Lk || D > most || v->size(3) > 2 * most) return none();
	diff_call c{*q, *k, *v, *lam, Tensor(), 0.0, 0, 0};
	key_mask  m;
	if(!mask_of(a[4], B, Lk, dev, m)) return none();
	if(a[4] != Py_None) {
		const Tensor& t = *tensor_of(a[4]);
		c.mask = t.dim() == 4 ? t.as_strided({t.size(0), Lk}, {t.stride(0), 1}) : t;
	}
	bool causal;
	if(!truth_of(a[5], causal) || !number_of(a[6], c.offset) || c.offset >= (int64_t)1 << 40 || c.offset <= -((int64_t)1 << 40)) return none();
	c.causal = causal;
	c.scale  = std::pow((double)D, -0.5);
	if(a[7] != Py_None && !real_of(a[7], c.scale)) return none();
	if(!((float)c.scale > 0.f && (float)c.scale < INFINITY) || has_tangent({q, k, v, lam})) return none();
	Tensor out;
	int    rc = AF3_OK;
	const bool graph = wants_grad({q, k, v, lam});
	if(graph && B * Hkv * ((Lk + 31) / 32) > 0xffffff) return none();   // (sizes whose gradients would be refused: the Python side says so)
	{
		without_gil g;
		if(graph) check_capture({q, k, v, lam}, dev), out = diff_function::apply(c.q, c.k, c.v, c.lam, given(c.mask), c.scale, c.causal, c.offset);
		else rc = c.forward(out, nullptr, nullptr, nullptr);
	}
	return answer(rc, std::move(out));
	END_HANDLE_TH_ERRORS
}

// check_capture(tensor or None...): raises where a gradient of these cannot be captured
PyObject* py_check_capture(PyObject*, PyObject* const* a, Py_ssize_t n) {
	HANDLE_TH_ERRORS
	std::vector<const Tensor*> tensors;
	int                        dev = -1;
	for(Py_ssize_t i = 0; i < n; i++)
		if(const Tensor* t = tensor_of(a[i]); t && t->is_cuda()) tensors.push_back(t), dev = (int)t->get_device();
	if(dev >= 0) check_capture(tensors, dev);
	return none();
	END_HANDLE_TH_ERRORS
}

#define AF3_FN(name, doc) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(py_##name)), METH_FASTCALL, doc}
PyMethodDef methods[] = {
	AF3_FN(attention, "attention(q, k, v, mask, bias, kernel_hint, exact_bias)"),
	AF3_FN(attention_fp8, "attention_fp8(q, k, v, mask, bias, compensated)"),
	AF3_FN(self_attention, "self_attention(x, mask, bias, wq, wk, wv, wg, q_bias, head, kernel_hint, exact_bias)"),
	AF3_FN(grid_kernel, "grid_kernel(pair, mask, bias, wq, wk, wv, wg, head)"),
	AF3_FN(grid_block, "grid_block(pair, ln_weight, ln_bias, eps, proj_weight, mask, wq, wk, wv, wg, out_proj, head, transpose, least_groups, kernel_hint, exact_bias)"),
	AF3_FN(out_projection, "out_projection(rows, out_proj)"),
	AF3_FN(linear, "linear(x, weight)"),
	AF3_FN(layernorm_pair_bias, "layernorm_pair_bias(pair, ln_weight, ln_bias, eps, proj_weight)"),
	AF3_FN(gated_linear_unit, "gated_linear_unit(x, weight, tag)"),
	AF3_FN(cross_attention, "cross_attention(q, k, v, mask, bias, scale)"),
	AF3_FN(position_bias, "position_bias(table, q_len, k_len, scheme, bidirectional, max_distance, q_positions, k_positions, q_offset)"),
	AF3_FN(rotary, "rotary(q, k, frequencies, positions, offset, interleaved, scale)"),
	AF3_FN(residual_norm, "residual_norm(x, y, weight, bias, gate, post_weight, norm, post_norm, sigmoid, residual_scale, eps)"),
	AF3_FN(differential_attention, "differential_attention(q, k, v, lam, mask, causal, q_offset, scale)"),
	AF3_FN(check_capture, "check_capture(tensor...): raises where their gradients cannot be captured into a graph"),
	AF3_FN(remember, "remember(tag, value, source...): a matrix derived from weights"),
	AF3_FN(recalls, "recalls(tag, source...): whether one is remembered for these"),
	AF3_FN(forget_source, "forget_source(address): drops what was derived from this tensor"),
	{"forget", py_forget, METH_NOARGS, "forget(): drops every remembered matrix"},
	{nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", "native host side of the entry points", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) {
	PyObject* m = PyModule_Create(&module);
	if(!m) return nullptr;
	for(auto& [name, value] : {std::pair<const char*, long>{"FUSED_WEIGHT", FUSED_WEIGHT}, {"Q_BIAS_ROW", Q_BIAS_ROW}, {"OUT_PROJ_T", OUT_PROJ_T}, {"GLU_T", GLU_T}}) PyModule_AddIntConstant(m, name, value);
	return m;
}
