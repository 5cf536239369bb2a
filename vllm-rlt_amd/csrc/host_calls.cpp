// Host side of the hot entry points: one C++ call from Python tensors to the C
// ABI.
//
// Checking a decode call's tensors, building its 29 C arguments and allocating
// its result in Python took 11 us of a 15 us call, twice what the kernel of a
// small batch runs.  The functions here do the same for the calls a serving
// loop makes: plain dense device tensors that pass every check.  Anything else
// (a failed check, a tensor subclass, an active function or dispatch mode, an
// empty batch) returns None before anything was done, and the caller takes
// the Python path, which raises the errors and handles the rest.  They return
// the result tensor, or the library's status when the launch was refused.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/TensorSubclassLikeUtils.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "rlt_kv.h"

namespace {

// Entry points of the library the Python package loaded (set by bind()).
decltype(&rlt_paged_decode) g_decode = nullptr;
decltype(&rlt_paged_decode_append) g_decode_append = nullptr;
decltype(&rlt_paged_decode_workspace_bytes) g_decode_bytes = nullptr;
decltype(&rlt_paged_prefill_split) g_prefill = nullptr;
decltype(&rlt_paged_prefill_split_workspace_bytes) g_prefill_bytes = nullptr;
decltype(&rlt_rope_kv_append) g_rope = nullptr;
decltype(&rlt_paged_decode_fp8) g_decode8 = nullptr;
decltype(&rlt_paged_decode_fp8_workspace_bytes) g_decode8_bytes = nullptr;
decltype(&rlt_paged_prefill_fp8) g_prefill8 = nullptr;
decltype(&rlt_paged_prefill_fp8_workspace_bytes) g_prefill8_bytes = nullptr;
decltype(&rlt_kv_append_fp8) g_append8 = nullptr;
decltype(&rlt_rope_axes_kv_append) g_rope_axes = nullptr;
decltype(&rlt_build_chunk_metadata) g_chunk_metadata = nullptr;
decltype(&rlt_paged_decode_int8) g_decode_i8 = nullptr;
decltype(&rlt_paged_decode_int8_workspace_bytes) g_decode_i8_bytes = nullptr;
decltype(&rlt_paged_prefill_int8) g_prefill_i8 = nullptr;
decltype(&rlt_paged_prefill_int8_workspace_bytes) g_prefill_i8_bytes = nullptr;
decltype(&rlt_kv_append_int8) g_append_i8 = nullptr;
decltype(&rlt_kv_gather_int8) g_gather_i8 = nullptr;

// A plain device tensor of torch.Tensor itself, or null.  (Parameters and other
// subclasses, wrappers of vmap / grad and fake tensors take the Python path.)
const at::Tensor* plain(PyObject* o) {
  if (Py_TYPE(o) != reinterpret_cast<PyTypeObject*>(THPVariableClass)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || at::isTensorSubclassLike(t)) return nullptr;
  return &t;
}

bool modes_active() {
  return at::impl::torch_function_mode_enabled() || c10::impl::TorchDispatchModeTLS::any_modes_set();
}

int code_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return RLT_FLOAT32;
    case at::kHalf: return RLT_FLOAT16;
    case at::kBFloat16: return RLT_BFLOAT16;
    default: return -1;
  }
}

bool aligned_rows(const at::Tensor& t) {
  if (t.stride(-1) != 1 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) return false;
  for (int64_t i = 0; i + 1 < t.dim(); ++i)
    if (t.stride(i) * t.element_size() % 16) return false;
  return true;
}

bool ints(const at::Tensor& t, at::ScalarType type) {
  return t.scalar_type() == type && t.dim() == 1 && t.is_contiguous();
}

// Layer-slice caches and q of one dtype and device: [blocks, page, kv heads, d]
// and [rows, heads, d].
bool attention_shapes(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& tables,
                      const at::Tensor& lens) {
  return q.dim() == 3 && k.dim() == 4 && k.sizes() == v.sizes() && k.strides() == v.strides() &&
         q.size(2) == k.size(3) && k.size(2) > 0 && q.size(1) > 0 && q.size(1) % k.size(2) == 0 &&
         code_of(q.scalar_type()) >= 0 && k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type() &&
         tables.scalar_type() == at::kInt && tables.dim() == 2 && tables.stride(1) == 1 && ints(lens, at::kInt) &&
         k.device() == q.device() && v.device() == q.device() && tables.device() == q.device() &&
         lens.device() == q.device();
}

// out when given and fitting (checked), a new tensor like q for None.
bool result_like(PyObject* o, const at::Tensor& q, at::Tensor* out) {
  if (o == Py_None) {
    *out = at::empty_like(q);
    return true;
  }
  const at::Tensor* t = plain(o);
  if (!t || t->sizes() != q.sizes() || t->scalar_type() != q.scalar_type() || t->device() != q.device()) return false;
  *out = *t;
  return true;
}

float scale_of(PyObject* o, int64_t d) {
  return static_cast<float>(o == Py_None ? 1.0 / std::sqrt(static_cast<double>(d)) : PyFloat_AS_DOUBLE(o));
}
bool scale_ok(PyObject* o) { return o == Py_None || PyFloat_CheckExact(o); }

PyObject* result(int rc, const at::Tensor& out) {
  if (rc != RLT_OK) return PyLong_FromLong(rc);
  return THPVariable_Wrap(out);
}

// decode(q, key, value, tables, lengths, out, workspace, scale, stream,
//        k_new, v_new, write_blocks, write_offsets, n_write); the last five
// absent for a decode without append, n_write None for all of write_blocks.
PyObject* decode(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if ((nargs != 9 && nargs != 14) || modes_active()) Py_RETURN_NONE;
  const at::Tensor* in[5];
  for (int i = 0; i < 5; ++i)
    if (!(in[i] = plain(args[i]))) Py_RETURN_NONE;
  const at::Tensor &q = *in[0], &k = *in[1], &v = *in[2], &tables = *in[3], &lens = *in[4];
  if (!attention_shapes(q, k, v, tables, lens) || !scale_ok(args[7]) || !PyLong_CheckExact(args[8])) Py_RETURN_NONE;
  const int64_t rows = q.size(0), hq = q.size(1), d = q.size(2), hkv = k.size(2);
  if (rows == 0 || tables.size(0) != rows || lens.size(0) != rows) Py_RETURN_NONE;
  const at::Tensor* app[4] = {};
  int64_t n = 0;
  if (nargs == 14) {
    for (int i = 0; i < 4; ++i)
      if (!(app[i] = plain(args[9 + i])) || app[i]->device() != q.device()) Py_RETURN_NONE;
    if (!ints(*app[2], at::kLong) || !ints(*app[3], at::kLong)) Py_RETURN_NONE;
    if (args[13] == Py_None) n = app[2]->size(0);
    else if (PyLong_CheckExact(args[13])) n = PyLong_AsLongLong(args[13]);
    else Py_RETURN_NONE;
    if (PyErr_Occurred()) {  // n_write past 64 bits
      PyErr_Clear();
      Py_RETURN_NONE;
    }
    if (n < 0 || n > rows || n > app[2]->size(0) || n > app[3]->size(0)) Py_RETURN_NONE;
    for (int i = 0; i < 2; ++i)
      if (app[i]->dim() != 3 || app[i]->size(1) != hkv || app[i]->size(2) != d || app[i]->size(0) < n ||
          app[i]->scalar_type() != q.scalar_type())
        Py_RETURN_NONE;
  }
  const int64_t need = g_decode_bytes(rows, hq, hkv, d);
  at::Tensor workspace, out;
  if (args[6] != Py_None) {
    const at::Tensor* w = plain(args[6]);
    if (!w || w->device() != q.device() || w->numel() * static_cast<int64_t>(w->element_size()) < need) Py_RETURN_NONE;
    workspace = *w;
  }
  if (!result_like(args[5], q, &out)) Py_RETURN_NONE;
  if (!workspace.defined()) workspace = at::empty({need}, q.options().dtype(at::kByte));
  void* const stream = PyLong_AsVoidPtr(args[8]);
  const int64_t nbytes = workspace.numel() * static_cast<int64_t>(workspace.element_size());
  const float scale = scale_of(args[7], d);
  const int code = code_of(q.scalar_type());
  int rc;
  Py_BEGIN_ALLOW_THREADS  // as ctypes does
  if (nargs == 14) {
    rc = g_decode_append(q.data_ptr(), q.strides().data(), k.data_ptr(), v.data_ptr(), k.strides().data(),
                         tables.data_ptr<int32_t>(), tables.stride(0), tables.size(1), lens.data_ptr<int32_t>(),
                         out.data_ptr(), out.strides().data(), rows, hq, hkv, d, k.size(1), k.size(0), scale, code,
                         app[0]->data_ptr(), app[0]->strides().data(), app[1]->data_ptr(), app[1]->strides().data(),
                         app[2]->data_ptr<int64_t>(), app[3]->data_ptr<int64_t>(), n, workspace.data_ptr(), nbytes,
                         stream);
  } else {
    rc = g_decode(q.data_ptr(), q.strides().data(), k.data_ptr(), v.data_ptr(), k.strides().data(),
                  tables.data_ptr<int32_t>(), tables.stride(0), tables.size(1), lens.data_ptr<int32_t>(),
                  out.data_ptr(), out.strides().data(), rows, hq, hkv, d, k.size(1), k.size(0), scale, code,
                  workspace.data_ptr(), nbytes, stream);
  }
  Py_END_ALLOW_THREADS
  return result(rc, out);
  END_HANDLE_TH_ERRORS
}

// Workspace bytes of a prefill; rows off 16 bytes take the per-token path, whose
// workspace is the fp32 one's.
int64_t prefill_need(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& tables,
                     const at::Tensor& out) {
  const bool rows16 = aligned_rows(q) && aligned_rows(out) && aligned_rows(k) && aligned_rows(v);
  return g_prefill_bytes(q.size(0), tables.size(0), tables.size(1), q.size(1), k.size(2), q.size(2), k.size(1),
                         rows16 ? code_of(q.scalar_type()) : int{RLT_FLOAT32});
}

// prefill_bytes(q, key, value, tables): what prefill() needs of a given workspace.
PyObject* prefill_bytes(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 4 || modes_active()) Py_RETURN_NONE;
  const at::Tensor* in[4];
  for (int i = 0; i < 4; ++i)
    if (!(in[i] = plain(args[i]))) Py_RETURN_NONE;
  const at::Tensor &q = *in[0], &k = *in[1], &v = *in[2], &tables = *in[3];
  if (q.dim() != 3 || k.dim() != 4 || v.dim() != 4 || tables.dim() != 2 || code_of(q.scalar_type()) < 0) Py_RETURN_NONE;
  return PyLong_FromLongLong(prefill_need(q, k, v, tables, q));
  END_HANDLE_TH_ERRORS
}

// prefill(q, key, value, tables, lengths, cu, max_seqlen_q, out, scale, stream,
//         workspace): the workspace for key segments or the per-token path is the
// given one when it is large enough, allocated here for None.
PyObject* prefill(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 11 || modes_active()) Py_RETURN_NONE;
  const at::Tensor* in[6];
  for (int i = 0; i < 6; ++i)
    if (!(in[i] = plain(args[i]))) Py_RETURN_NONE;
  const at::Tensor &q = *in[0], &k = *in[1], &v = *in[2], &tables = *in[3], &lens = *in[4], &cu = *in[5];
  if (!attention_shapes(q, k, v, tables, lens) || !ints(cu, at::kInt) || cu.device() != q.device() ||
      !PyLong_CheckExact(args[6]) || !scale_ok(args[8]) || !PyLong_CheckExact(args[9]))
    Py_RETURN_NONE;
  const int64_t total = q.size(0), hq = q.size(1), d = q.size(2), hkv = k.size(2), nseq = tables.size(0);
  if (total == 0 || nseq == 0 || lens.size(0) != nseq || cu.size(0) != nseq + 1) Py_RETURN_NONE;
  const int64_t max_q = PyLong_AsLongLong(args[6]);
  if (max_q == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  at::Tensor out;
  if (!result_like(args[7], q, &out)) Py_RETURN_NONE;
  const int code = code_of(q.scalar_type());
  const int64_t need = prefill_need(q, k, v, tables, out);
  at::Tensor workspace;
  if (args[10] != Py_None) {
    const at::Tensor* w = plain(args[10]);
    if (!w || w->scalar_type() != at::kByte || w->device() != q.device() || w->numel() < need) Py_RETURN_NONE;
    workspace = *w;
  } else {
    workspace = at::empty({need > 0 ? need : 1}, q.options().dtype(at::kByte));
  }
  void* const stream = PyLong_AsVoidPtr(args[9]);
  const float scale = scale_of(args[8], d);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = g_prefill(q.data_ptr(), q.strides().data(), k.data_ptr(), v.data_ptr(), k.strides().data(),
                 tables.data_ptr<int32_t>(), tables.stride(0), tables.size(1), lens.data_ptr<int32_t>(),
                 cu.data_ptr<int32_t>(), nseq, total, max_q, out.data_ptr(), out.strides().data(), hq, hkv, d, k.size(1),
                 k.size(0), scale, code, workspace.data_ptr(), workspace.numel(), stream);
  Py_END_ALLOW_THREADS
  return result(rc, out);
  END_HANDLE_TH_ERRORS
}

// rope(key_cache, value_cache, layer, write_blocks, write_offsets, q, k, v, cos,
//      sin, out, n_rows, stream); cos and sin [rows, d].
PyObject* rope(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 13 || modes_active() || !PyLong_CheckExact(args[2]) || !PyLong_CheckExact(args[12])) Py_RETURN_NONE;
  static constexpr int kAt[9] = {0, 1, 3, 4, 5, 6, 7, 8, 9};
  const at::Tensor* in[9];
  for (int i = 0; i < 9; ++i)
    if (!(in[i] = plain(args[kAt[i]])) || in[i]->device() != in[0]->device()) Py_RETURN_NONE;
  const at::Tensor &kc = *in[0], &vc = *in[1], &wb = *in[2], &wo = *in[3], &q = *in[4], &k = *in[5], &v = *in[6],
                   &cos = *in[7], &sin = *in[8];
  if (kc.dim() != 5 || kc.sizes() != vc.sizes() || kc.strides() != vc.strides() || q.dim() != 3) Py_RETURN_NONE;
  const int64_t hkv = kc.size(3), d = kc.size(4), rows = q.size(0);
  const int code = code_of(kc.scalar_type());
  if (code < 0 || hkv == 0 || d % 2 || q.size(2) != d || q.size(1) % hkv || !ints(wb, at::kLong) || !ints(wo, at::kLong))
    Py_RETURN_NONE;
  for (const at::Tensor* t : {&k, &v})
    if (t->dim() != 3 || t->size(0) != rows || t->size(1) != hkv || t->size(2) != d) Py_RETURN_NONE;
  for (const at::Tensor* t : {&cos, &sin})
    if (t->dim() != 2 || t->size(0) != rows || t->size(1) != d) Py_RETURN_NONE;
  for (const at::Tensor* t : {&vc, &q, &k, &v, &cos, &sin})
    if (t->scalar_type() != kc.scalar_type()) Py_RETURN_NONE;
  if (cos.strides() != sin.strides()) Py_RETURN_NONE;
  int64_t n = wb.size(0);
  if (args[11] != Py_None) {
    if (!PyLong_CheckExact(args[11])) Py_RETURN_NONE;
    n = PyLong_AsLongLong(args[11]);
  }
  const int64_t layer = PyLong_AsLongLong(args[2]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  if (n < 0 || n > wb.size(0) || n > wo.size(0) || n > rows) Py_RETURN_NONE;
  at::Tensor out;
  if (!result_like(args[10], q, &out)) Py_RETURN_NONE;
  void* const stream = PyLong_AsVoidPtr(args[12]);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = g_rope(kc.data_ptr(), vc.data_ptr(), kc.strides().data(), q.data_ptr(), q.strides().data(), k.data_ptr(),
              k.strides().data(), v.data_ptr(), v.strides().data(), cos.data_ptr(), sin.data_ptr(), cos.strides().data(),
              out.data_ptr(), out.strides().data(), wb.data_ptr<int64_t>(), wo.data_ptr<int64_t>(), rows, n, layer,
              kc.size(1), kc.size(0), kc.size(2), q.size(1), hkv, d, code, stream);
  Py_END_ALLOW_THREADS
  return result(rc, out);
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------- 8-bit KV caches
// Whether t is on the current device, which a launch goes to.
bool here(const at::Tensor& t) {
  static const c10::impl::VirtualGuardImpl device(c10::DeviceType::CUDA);
  return t.device().index() == device.getDevice().index();
}

// All of args[at[0]], args[at[1]], ... plain tensors of the current device.
template <int N>
bool all_plain(PyObject* const* args, const int (&at)[N], const at::Tensor* (&out)[N]) {
  for (int i = 0; i < N; ++i)
    if (!(out[i] = plain(args[at[i]])) || out[i]->device() != out[0]->device()) return false;
  return here(*out[0]);
}

// An int64 argument; false where it is none (a subclass, or past 64 bits).
bool int_of(PyObject* o, int64_t* x) {
  if (!PyLong_CheckExact(o)) return false;
  int overflow = 0;
  *x = PyLong_AsLongLongAndOverflow(o, &overflow);
  return !overflow;
}

// e4m3 codes of dims dims with e8m0 scales of the same shape without the last.
bool cache8(const at::Tensor& k, const at::Tensor& v, const at::Tensor& ks, const at::Tensor& vs, int64_t dims) {
  return k.dim() == dims && k.scalar_type() == at::kFloat8_e4m3fn && v.scalar_type() == at::kFloat8_e4m3fn &&
         ks.scalar_type() == at::kFloat8_e8m0fnu && vs.scalar_type() == at::kFloat8_e8m0fnu && k.sizes() == v.sizes() &&
         k.strides() == v.strides() && ks.sizes() == k.sizes().slice(0, dims - 1) && vs.sizes() == ks.sizes() &&
         vs.strides() == ks.strides();
}

// Signed codes of dims dims with fp32 scales, one a block (and layer) and head.
bool cache_i8(const at::Tensor& k, const at::Tensor& v, const at::Tensor& ks, const at::Tensor& vs, int64_t dims) {
  if (k.dim() != dims || k.scalar_type() != at::kChar || v.scalar_type() != at::kChar || ks.scalar_type() != at::kFloat ||
      vs.scalar_type() != at::kFloat || k.sizes() != v.sizes() || k.strides() != v.strides() || ks.dim() != dims - 2 ||
      vs.sizes() != ks.sizes() || vs.strides() != ks.strides())
    return false;
  for (int64_t i = 0; i < dims - 3; ++i)
    if (ks.size(i) != k.size(i)) return false;
  return ks.size(dims - 3) == k.size(dims - 2);
}

// Which of the two caches a call is over, its check and its entry points.
struct Form8 {
  bool (*cache)(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, int64_t);
  decltype(g_decode8)*decode;
  decltype(g_decode8_bytes)*decode_bytes;
  decltype(g_prefill8)*prefill;
  decltype(g_prefill8_bytes)*prefill_bytes;
  decltype(g_append8)*append;
};
const Form8 kFp8 = {cache8, &g_decode8, &g_decode8_bytes, &g_prefill8, &g_prefill8_bytes, &g_append8};
const Form8 kInt8 = {cache_i8, &g_decode_i8, &g_decode_i8_bytes, &g_prefill_i8, &g_prefill_i8_bytes, &g_append_i8};

// What decode and prefill share: q, cache, tables and lengths in args[0 .. 6].
bool attention8(const Form8& form, const at::Tensor* const* in) {
  const at::Tensor &q = *in[0], &k = *in[1], &tables = *in[5], &lens = *in[6];
  return form.cache(k, *in[2], *in[3], *in[4], 4) && q.dim() == 3 && q.size(2) == k.size(3) && code_of(q.scalar_type()) >= 0 &&
         k.size(2) > 0 && q.size(1) > 0 && q.size(1) % k.size(2) == 0 && q.size(0) > 0 && tables.scalar_type() == at::kInt &&
         tables.dim() == 2 && tables.stride(1) == 1 && tables.size(0) > 0 && ints(lens, at::kInt) && lens.size(0) == tables.size(0);
}

// The workspace given in o if it holds need contiguous bytes on q's device, a new one for None.
bool workspace_of(PyObject* o, int64_t need, const at::Tensor& q, at::Tensor* ws) {
  if (o == Py_None) {
    *ws = at::empty({need}, q.options().dtype(at::kByte));
    return true;
  }
  const at::Tensor* w = plain(o);
  if (!w || w->device() != q.device() || !w->is_contiguous() || w->numel() * static_cast<int64_t>(w->element_size()) < need)
    return false;
  *ws = *w;
  return true;
}

// decode8(q, key, value, key_scales, value_scales, tables, lengths, out, workspace, scale, stream)
PyObject* decode8(const Form8& form, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  static constexpr int kAt[7] = {0, 1, 2, 3, 4, 5, 6};
  const at::Tensor* in[7];
  if (nargs != 11 || modes_active() || !all_plain(args, kAt, in) || !attention8(form, in) || !scale_ok(args[9])) Py_RETURN_NONE;
  const at::Tensor &q = *in[0], &k = *in[1], &tables = *in[5];
  const int64_t rows = q.size(0), hq = q.size(1), d = q.size(2), hkv = k.size(2), width = tables.size(1);
  if (tables.size(0) != rows) Py_RETURN_NONE;
  at::Tensor out, ws;
  if (!workspace_of(args[8], (*form.decode_bytes)(rows, width, hq, hkv, d, k.size(1)), q, &ws) || !result_like(args[7], q, &out))
    Py_RETURN_NONE;
  void* const stream = PyLong_AsVoidPtr(args[10]);
  const float scale = scale_of(args[9], d);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = (*form.decode)(q.data_ptr(), q.strides().data(), k.data_ptr(), in[2]->data_ptr(), k.strides().data(), in[3]->data_ptr(),
                 in[4]->data_ptr(), in[3]->strides().data(), tables.data_ptr<int32_t>(), tables.stride(0), width,
                 in[6]->data_ptr<int32_t>(), out.data_ptr(), out.strides().data(), rows, hq, hkv, d, k.size(1), k.size(0),
                 scale, code_of(q.scalar_type()), ws.data_ptr(), ws.numel() * static_cast<int64_t>(ws.element_size()), stream);
  Py_END_ALLOW_THREADS
  return result(rc, out);
  END_HANDLE_TH_ERRORS
}

// prefill8(q, key, value, key_scales, value_scales, tables, lengths, cu, max_seqlen_q, out, workspace,
//          scale, batch_invariant, stream)
PyObject* prefill8(const Form8& form, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  static constexpr int kAt[8] = {0, 1, 2, 3, 4, 5, 6, 7};
  const at::Tensor* in[8];
  int64_t longest;
  if (nargs != 14 || modes_active() || !all_plain(args, kAt, in) || !attention8(form, in) || !scale_ok(args[11]) ||
      !PyBool_Check(args[12]) || !int_of(args[8], &longest))
    Py_RETURN_NONE;
  const at::Tensor &q = *in[0], &k = *in[1], &tables = *in[5], &cu = *in[7];
  const int64_t total = q.size(0), hq = q.size(1), d = q.size(2), hkv = k.size(2), n = tables.size(0), width = tables.size(1);
  if (!ints(cu, at::kInt) || cu.size(0) != n + 1) Py_RETURN_NONE;
  const int64_t need = args[12] == Py_True ? 0 : (*form.prefill_bytes)(total, n, width, hq, hkv, d, k.size(1));
  at::Tensor out, ws;
  if (!workspace_of(args[10], need, q, &ws) || !result_like(args[9], q, &out)) Py_RETURN_NONE;
  void* const stream = PyLong_AsVoidPtr(args[13]);
  const float scale = scale_of(args[11], d);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = (*form.prefill)(q.data_ptr(), q.strides().data(), k.data_ptr(), in[2]->data_ptr(), k.strides().data(), in[3]->data_ptr(),
                  in[4]->data_ptr(), in[3]->strides().data(), tables.data_ptr<int32_t>(), tables.stride(0), width,
                  in[6]->data_ptr<int32_t>(), cu.data_ptr<int32_t>(), n, total, longest, out.data_ptr(), out.strides().data(),
                  hq, hkv, d, k.size(1), k.size(0), scale, code_of(q.scalar_type()), need ? ws.data_ptr() : nullptr,
                  ws.numel() * static_cast<int64_t>(ws.element_size()), stream);
  Py_END_ALLOW_THREADS
  return result(rc, out);
  END_HANDLE_TH_ERRORS
}

// Rows to write: o, or all of write_blocks for None; false where they are not covered.
bool rows_of(PyObject* o, const at::Tensor& wb, const at::Tensor& wo, int64_t rows, int64_t* n) {
  *n = wb.size(0);
  return (o == Py_None || int_of(o, n)) && *n >= 0 && *n <= wb.size(0) && *n <= wo.size(0) && *n <= rows;
}

// append8(key_cache, value_cache, key_scales, value_scales, layer, write_blocks, write_offsets, k, v, n_rows,
//         stream): an int, the library's status.
PyObject* append8(const Form8& form, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  static constexpr int kAt[8] = {0, 1, 2, 3, 5, 6, 7, 8};
  const at::Tensor* in[8];
  int64_t layer, n;
  if (nargs != 11 || modes_active() || !all_plain(args, kAt, in) || !int_of(args[4], &layer)) Py_RETURN_NONE;
  const at::Tensor &kc = *in[0], &wb = *in[4], &wo = *in[5], &k = *in[6], &v = *in[7];
  if (!form.cache(kc, *in[1], *in[2], *in[3], 5) || !ints(wb, at::kLong) || !ints(wo, at::kLong) || k.dim() != 3 || v.dim() != 3 ||
      code_of(k.scalar_type()) < 0 || v.scalar_type() != k.scalar_type())
    Py_RETURN_NONE;
  const int64_t hkv = kc.size(3), d = kc.size(4);
  for (const at::Tensor* t : {&k, &v})
    if (t->size(1) != hkv || t->size(2) != d) Py_RETURN_NONE;
  if (!rows_of(args[9], wb, wo, std::min(k.size(0), v.size(0)), &n)) Py_RETURN_NONE;
  void* const stream = PyLong_AsVoidPtr(args[10]);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = (*form.append)(kc.data_ptr(), in[1]->data_ptr(), kc.strides().data(), in[2]->data_ptr(), in[3]->data_ptr(),
                 in[2]->strides().data(), k.data_ptr(), k.strides().data(), v.data_ptr(), v.strides().data(),
                 wb.data_ptr<int64_t>(), wo.data_ptr<int64_t>(), n, layer, kc.size(1), kc.size(0), kc.size(2), hkv, d,
                 code_of(k.scalar_type()), stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
  END_HANDLE_TH_ERRORS
}

// gather_i8(key_cache, value_cache, key_scales, value_scales, layer, blocks, offsets, dtype code, n_rows, stream): (k, v)
PyObject* gather_i8(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  static constexpr int kAt[6] = {0, 1, 2, 3, 5, 6};
  const at::Tensor* in[6];
  int64_t layer, code, n;
  if (nargs != 10 || modes_active() || !all_plain(args, kAt, in) || !int_of(args[4], &layer) || !int_of(args[7], &code)) Py_RETURN_NONE;
  const at::Tensor &kc = *in[0], &blocks = *in[4], &offsets = *in[5];
  if (!cache_i8(kc, *in[1], *in[2], *in[3], 5) || !ints(blocks, at::kLong) || !ints(offsets, at::kLong)) Py_RETURN_NONE;
  if (!rows_of(args[8], blocks, offsets, blocks.size(0), &n)) Py_RETURN_NONE;
  const at::ScalarType type = code == RLT_FLOAT32 ? at::kFloat : code == RLT_FLOAT16 ? at::kHalf : at::kBFloat16;
  const at::Tensor k = at::empty({n, kc.size(3), kc.size(4)}, kc.options().dtype(type)), v = at::empty_like(k);
  void* const stream = PyLong_AsVoidPtr(args[9]);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = g_gather_i8(kc.data_ptr(), in[1]->data_ptr(), kc.strides().data(), in[2]->data_ptr(), in[3]->data_ptr(),
                   in[2]->strides().data(), blocks.data_ptr<int64_t>(), offsets.data_ptr<int64_t>(), n, k.data_ptr(), v.data_ptr(),
                   layer, kc.size(1), kc.size(0), kc.size(2), kc.size(3), kc.size(4), static_cast<int>(code), stream);
  Py_END_ALLOW_THREADS
  if (rc != RLT_OK) return PyLong_FromLong(rc);
  PyObject* const pair = PyTuple_New(2);
  if (!pair) return nullptr;
  PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(k));
  PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(v));
  return pair;
  END_HANDLE_TH_ERRORS
}

template <PyObject* (*F)(const Form8&, PyObject* const*, Py_ssize_t), const Form8& FORM>
PyObject* of_form(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return F(FORM, args, nargs);
}

// rope_axes(key_cache, value_cache, layer, write_blocks, write_offsets, q, k, v, positions, table, axes,
//           key_scales, value_scales, out, n_rows, stream); axes a tuple of ints, scales None for a cache of q's type.
PyObject* rope_axes(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  static constexpr int kAt[9] = {0, 1, 3, 4, 5, 6, 7, 8, 9};
  const at::Tensor* in[9];
  int64_t layer, n;
  if (nargs != 16 || modes_active() || !all_plain(args, kAt, in) || !int_of(args[2], &layer) || !PyTuple_CheckExact(args[10]))
    Py_RETURN_NONE;
  const at::Tensor &kc = *in[0], &vc = *in[1], &wb = *in[2], &wo = *in[3], &q = *in[4], &k = *in[5], &v = *in[6],
                   &pos = *in[7], &table = *in[8];
  const at::Tensor *ks = nullptr, *vs = nullptr;
  if (args[11] != Py_None || args[12] != Py_None) {
    if (!(ks = plain(args[11])) || !(vs = plain(args[12])) || ks->device() != q.device() || vs->device() != q.device() ||
        !cache8(kc, vc, *ks, *vs, 5))
      Py_RETURN_NONE;
  } else if (kc.dim() != 5 || kc.sizes() != vc.sizes() || kc.strides() != vc.strides() || kc.scalar_type() != q.scalar_type() ||
             vc.scalar_type() != q.scalar_type()) {
    Py_RETURN_NONE;
  }
  const int64_t hkv = kc.size(3), d = kc.size(4), rows = q.size(0);
  if (q.dim() != 3 || code_of(q.scalar_type()) < 0 || hkv == 0 || q.size(2) != d || q.size(1) == 0 || q.size(1) % hkv ||
      !ints(wb, at::kLong) || !ints(wo, at::kLong))
    Py_RETURN_NONE;
  for (const at::Tensor* t : {&k, &v})
    if (t->dim() != 3 || t->size(0) != rows || t->size(1) != hkv || t->size(2) != d || t->scalar_type() != q.scalar_type())
      Py_RETURN_NONE;
  if (pos.scalar_type() != at::kLong || pos.dim() != 2 || pos.size(0) != rows || table.scalar_type() != at::kFloat ||
      table.dim() != 3 || table.size(2) != 2 || !table.is_contiguous())
    Py_RETURN_NONE;
  constexpr int64_t kMost = 256;
  const int64_t half = table.size(1);
  if (half > kMost || 2 * half > d || PyTuple_GET_SIZE(args[10]) != half) Py_RETURN_NONE;
  uint8_t axes[kMost];
  for (int64_t j = 0; j < half; ++j) {
    int64_t x;
    if (!int_of(PyTuple_GET_ITEM(args[10], j), &x) || x < 0 || x > 255) Py_RETURN_NONE;
    axes[j] = static_cast<uint8_t>(x);
  }
  at::Tensor out;
  if (!rows_of(args[14], wb, wo, rows, &n) || !result_like(args[13], q, &out)) Py_RETURN_NONE;
  void* const stream = PyLong_AsVoidPtr(args[15]);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = g_rope_axes(kc.data_ptr(), vc.data_ptr(), kc.strides().data(), ks ? ks->data_ptr() : nullptr,
                   vs ? vs->data_ptr() : nullptr, ks ? ks->strides().data() : nullptr, q.data_ptr(), q.strides().data(),
                   k.data_ptr(), k.strides().data(), v.data_ptr(), v.strides().data(), out.data_ptr(), out.strides().data(),
                   pos.data_ptr<int64_t>(), pos.strides().data(), pos.size(1), table.data_ptr<float>(), table.size(0), axes,
                   half, wb.data_ptr<int64_t>(), wo.data_ptr<int64_t>(), rows, n, layer, kc.size(1), kc.size(0), kc.size(2),
                   q.size(1), hkv, d, code_of(q.scalar_type()), stream);
  Py_END_ALLOW_THREADS
  return result(rc, out);
  END_HANDLE_TH_ERRORS
}

// chunk_metadata(descriptors, count, size, tables, page, cu, lengths, positions, sequences, blocks, offsets,
//                out_tables, out_width, stream): an int, the library's status.
PyObject* chunk_metadata(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  static constexpr int kAt[9] = {0, 3, 5, 6, 7, 8, 9, 10, 11};
  const at::Tensor* in[9];
  int64_t count, size, page, width;
  if (nargs != 14 || modes_active() || !int_of(args[1], &count) || !int_of(args[2], &size) || !int_of(args[4], &page) ||
      !int_of(args[12], &width))
    Py_RETURN_NONE;
  PyObject* const d0 = args[0];
  if (Py_TYPE(d0) != reinterpret_cast<PyTypeObject*>(THPVariableClass)) Py_RETURN_NONE;
  const at::Tensor& desc = THPVariable_Unpack(d0);
  if (!desc.defined() || desc.layout() != at::kStrided || at::isTensorSubclassLike(desc)) Py_RETURN_NONE;
  for (int i = 1; i < 9; ++i)
    if (!(in[i] = plain(args[kAt[i]])) || in[i]->device() != in[1]->device()) Py_RETURN_NONE;
  if (!here(*in[1])) Py_RETURN_NONE;
  const at::Tensor &tables = *in[1], &cu = *in[2], &lens = *in[3], &out = *in[8];
  if (desc.is_cuda() ? desc.device() != tables.device() : !desc.device().is_cpu() || !desc.is_pinned()) Py_RETURN_NONE;
  if (desc.scalar_type() != at::kLong || desc.dim() != 2 || desc.size(1) != 4 || !desc.is_contiguous() ||
      tables.scalar_type() != at::kInt || tables.dim() != 3 || !tables.is_contiguous() || out.scalar_type() != at::kInt ||
      out.dim() != 2 || out.stride(1) != 1 || !ints(cu, at::kInt) || !ints(lens, at::kInt))
    Py_RETURN_NONE;
  const int64_t capacity = in[4]->numel();
  for (int i = 4; i < 8; ++i)
    if (!ints(*in[i], at::kLong) || in[i]->numel() != capacity) Py_RETURN_NONE;
  if (count < 0 || count > size || count > desc.size(0) || size > cu.size(0) - 1 || size > lens.size(0) || size > out.size(0) ||
      width < 0 || width > tables.size(2) || width > out.size(1))
    Py_RETURN_NONE;
  void* const stream = PyLong_AsVoidPtr(args[13]);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = g_chunk_metadata(desc.data_ptr<int64_t>(), count, size, tables.data_ptr<int32_t>(), tables.size(0), tables.size(2),
                        tables.size(1), page, cu.data_ptr<int32_t>(), lens.data_ptr<int32_t>(), in[4]->data_ptr<int64_t>(),
                        in[5]->data_ptr<int64_t>(), in[6]->data_ptr<int64_t>(), in[7]->data_ptr<int64_t>(), capacity,
                        out.data_ptr<int32_t>(), size > 1 ? out.stride(0) : width, width, stream);  // one row's stride is nobody's
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
  END_HANDLE_TH_ERRORS
}

// bind(addresses of the loaded library's entry points, in HOST_CALLED's order).
template <typename F>
bool bind_one(PyObject* o, F* f) {
  void* const p = PyLong_AsVoidPtr(o);
  if (!p && PyErr_Occurred()) return false;
  *f = reinterpret_cast<F>(p);
  return true;
}
PyObject* bind(PyObject*, PyObject* args) {
  PyObject* a[19];
  if (!PyArg_ParseTuple(args, "OOOOOOOOOOOOOOOOOOO", &a[0], &a[1], &a[2], &a[3], &a[4], &a[5], &a[6], &a[7], &a[8], &a[9], &a[10],
                        &a[11], &a[12], &a[13], &a[14], &a[15], &a[16], &a[17], &a[18]))
    return nullptr;
  if (!bind_one(a[0], &g_decode) || !bind_one(a[1], &g_decode_append) || !bind_one(a[2], &g_decode_bytes) ||
      !bind_one(a[3], &g_prefill) || !bind_one(a[4], &g_prefill_bytes) || !bind_one(a[5], &g_rope) ||
      !bind_one(a[6], &g_decode8) || !bind_one(a[7], &g_decode8_bytes) || !bind_one(a[8], &g_prefill8) ||
      !bind_one(a[9], &g_prefill8_bytes) || !bind_one(a[10], &g_append8) || !bind_one(a[11], &g_rope_axes) ||
      !bind_one(a[12], &g_chunk_metadata) || !bind_one(a[13], &g_decode_i8) || !bind_one(a[14], &g_decode_i8_bytes) ||
      !bind_one(a[15], &g_prefill_i8) || !bind_one(a[16], &g_prefill_i8_bytes) || !bind_one(a[17], &g_append_i8) ||
      !bind_one(a[18], &g_gather_i8))
    return nullptr;
  Py_RETURN_NONE;
}

PyMethodDef kMethods[] = {
    {"bind", bind, METH_VARARGS, nullptr},
    {"decode", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(decode)), METH_FASTCALL, nullptr},
    {"prefill", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(prefill)), METH_FASTCALL, nullptr},
    {"prefill_bytes", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(prefill_bytes)), METH_FASTCALL, nullptr},
    {"rope", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rope)), METH_FASTCALL, nullptr},
    {"decode8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(of_form<decode8, kFp8>)), METH_FASTCALL, nullptr},
    {"decode_i8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(of_form<decode8, kInt8>)), METH_FASTCALL, nullptr},
    {"prefill8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(of_form<prefill8, kFp8>)), METH_FASTCALL, nullptr},
    {"prefill_i8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(of_form<prefill8, kInt8>)), METH_FASTCALL, nullptr},
    {"append8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(of_form<append8, kFp8>)), METH_FASTCALL, nullptr},
    {"append_i8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(of_form<append8, kInt8>)), METH_FASTCALL, nullptr},
    {"rope_axes", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rope_axes)), METH_FASTCALL, nullptr},
    {"chunk_metadata", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(chunk_metadata)), METH_FASTCALL, nullptr},
    {"gather_i8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(gather_i8)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_host_calls", nullptr, -1, kMethods};

}  // namespace

PyMODINIT_FUNC PyInit__host_calls(void) { return PyModule_Create(&kModule); }
