// CPython module harpq_b200_bind: the serving operators' calls from torch tensors to the C ABI.
//
// A step's smallest calls take a few microseconds on the GPU, less than checking a dozen tensors
// through Python attributes.  Each function here checks its tensors, fills the argument structure
// and calls the C entry point with the tensors' device current (it launches on the current one); it
// returns that call's status, or -1 without calling where an argument does not fit, and the Python
// method then says which.
#include <Python.h>

#include <ATen/MemoryOverlap.h>
#include <c10/core/DeviceGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "harpq_b200.h"

namespace {

using at::Tensor;

constexpr long kUnfit = -1;

const Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

// An int32 tensor of n elements on GPU `device`; None gives nullptr where `optional`.
bool ints(PyObject* o, int64_t n, int device, bool optional, const int32_t** at) {
  *at = nullptr;
  if (o == Py_None) return optional;
  const Tensor* t = tensor(o);
  if (t == nullptr || t->scalar_type() != at::kInt || t->numel() != n || !t->is_contiguous() || !t->is_cuda() ||
      t->get_device() != device)
    return false;
  *at = static_cast<const int32_t*>(t->const_data_ptr());
  return true;
}

int code(at::ScalarType t) { return t == at::kFloat ? HQB_F32 : t == at::kHalf ? HQB_F16 : t == at::kBFloat16 ? HQB_BF16 : -1; }

// [rows][heads][dim] with adjacent elements in a head.
bool heads(PyObject* o, int64_t rows, int64_t heads, int64_t dim, int type, int device, const Tensor** t) {
  *t = tensor(o);
  return *t != nullptr && (*t)->dim() == 3 && (rows < 0 || (*t)->size(0) == rows) && (*t)->size(1) == heads &&
         (*t)->size(2) == dim && (type < 0 || code((*t)->scalar_type()) == type) && (*t)->is_cuda() &&
         (*t)->get_device() == device && (dim == 1 || (*t)->stride(2) == 1);
}

// Whether each element of a result has a place of its own.
bool distinct(const Tensor& t) { return at::has_internal_overlap(t) != at::MemOverlap::Yes; }

// The current stream of the device, or the one given as a number.
void* stream_of(PyObject* o, int device) {
  if (o == Py_None) return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream();
  return PyLong_AsVoidPtr(o);
}

PyObject* status(long s) { return PyLong_FromLong(s); }

// Makes GPU `device` current until the end of the scope: of two GPUs' default streams, both handle 0,
// a launch takes the current one's.
class OnDevice {
 public:
  explicit OnDevice(int device) {
    const c10::Device d(c10::kCUDA, static_cast<c10::DeviceIndex>(device));
    if (c10::impl::getDeviceGuardImpl(c10::kCUDA)->getDevice() != d) guard_.reset_device(d);
  }

 private:
  c10::OptionalDeviceGuard guard_;
};

// page_plan(args address, device, stream, context_lens, new_lens, held, tables, free_pages, free_head,
//           parents, slots, held_out, free_head_out, mask, words)
// The structure at args has the plan's sizes and output addresses; the last five are outputs that
// some calls leave out.
PyObject* page_plan(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 15) return status(kUnfit);
  auto* p = static_cast<hqb_page_plan_args*>(PyLong_AsVoidPtr(a[0]));
  const int device = static_cast<int>(PyLong_AsLong(a[1]));
  const OnDevice on(device);
  const Tensor* table = nullptr;
  const int32_t* rows = nullptr;
  if (!ints(a[3], p->requests, device, false, &p->context_lens) || !ints(a[4], p->requests, device, false, &p->new_lens) ||
      !ints(a[5], p->requests, device, true, &p->held))
    return status(kUnfit);
  p->tables = nullptr;
  p->free_pages = p->free_head = nullptr;
  p->table_stride = p->free_count = 0;
  p->slots = p->held_out = p->free_head_out = nullptr;
  if (a[6] != Py_None) {
    const Tensor* pool = a[7] == Py_None ? nullptr : tensor(a[7]);
    table = tensor(a[6]);
    if (pool == nullptr || table == nullptr || table->dim() != 2 || table->size(0) != p->requests ||
        !ints(a[6], table->numel(), device, false, &rows) || !ints(a[7], pool->numel(), device, false, &p->free_pages) ||
        !ints(a[8], 1, device, false, &p->free_head))
      return status(kUnfit);
    p->tables = const_cast<int32_t*>(rows);
    p->table_stride = static_cast<uint32_t>(table->size(1));
    p->free_count = static_cast<uint32_t>(pool->numel());
    p->slots = static_cast<int32_t*>(PyLong_AsVoidPtr(a[10]));
    p->held_out = static_cast<int32_t*>(PyLong_AsVoidPtr(a[11]));
    p->free_head_out = static_cast<int32_t*>(PyLong_AsVoidPtr(a[12]));
  }
  p->parents = nullptr;
  p->mask = nullptr;
  p->mask_words = p->parent_count = 0;
  if (a[9] != Py_None) {
    const Tensor* tree = tensor(a[9]);
    p->mask_words = static_cast<uint32_t>(PyLong_AsUnsignedLong(a[14]));
    if (tree == nullptr || p->mask_words == 0 || !ints(a[9], tree->numel(), device, false, &p->parents) ||
        tree->numel() > INT32_MAX)
      return status(kUnfit);
    p->parent_count = static_cast<uint32_t>(tree->numel());
    if (p->parent_count == 0) p->parents = p->starts;  // none is read: a step without tokens
    p->mask = static_cast<uint32_t*>(PyLong_AsVoidPtr(a[13]));
  }
  return status(hqb_page_plan(p, stream_of(a[2], device)));
}

// cache_append(cache address, device, stream, k, v, slots, rows, flags address)
PyObject* cache_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 8) return status(kUnfit);
  const auto* c = static_cast<const hqb_paged_cache*>(PyLong_AsVoidPtr(a[0]));
  const int device = static_cast<int>(PyLong_AsLong(a[1]));
  const OnDevice on(device);
  const Tensor *k, *v, *slots = tensor(a[5]);
  if (slots == nullptr || !heads(a[3], -1, c->kv_heads, c->head_dim, -1, device, &k) ||
      !heads(a[4], k->size(0), c->kv_heads, c->head_dim, code(k->scalar_type()), device, &v) || k->strides() != v->strides() ||
      code(k->scalar_type()) < 0)
    return status(kUnfit);
  const int64_t count = slots->numel();
  const int32_t *to, *pick;
  if (!ints(a[5], count, device, false, &to) || !ints(a[6], count, device, true, &pick) || (pick == nullptr && count > k->size(0)))
    return status(kUnfit);
  return status(hqb_cache_append(c, k->const_data_ptr(), v->const_data_ptr(), code(k->scalar_type()),
                                 static_cast<uint64_t>(k->stride(0)), static_cast<uint64_t>(k->stride(1)),
                                 static_cast<uint32_t>(k->size(0)), pick, to, static_cast<uint32_t>(count),
                                 static_cast<int*>(PyLong_AsVoidPtr(a[7])), stream_of(a[2], device)));
}

// tree_attention(cache address, args address, workspace address, workspace bytes, device, stream, q, k, v,
//                tables, context_lens, starts, mask, scale, out, lse)
// The structure at args has max_new, max_context and q_heads, and in requests and tokens the most
// that the workspace was made for.
PyObject* tree_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 16) return status(kUnfit);
  const auto* c = static_cast<const hqb_paged_cache*>(PyLong_AsVoidPtr(a[0]));
  hqb_attention_args p = *static_cast<const hqb_attention_args*>(PyLong_AsVoidPtr(a[1]));
  const int device = static_cast<int>(PyLong_AsLong(a[4]));
  const OnDevice on(device);
  const Tensor *q, *k, *v, *out, *table = tensor(a[9]), *ctx = tensor(a[10]);
  if (ctx == nullptr || table == nullptr || !heads(a[6], -1, p.q_heads, c->head_dim, c->dtype, device, &q)) return status(kUnfit);
  const int64_t tokens = q->size(0), requests = ctx->numel();
  if (tokens > p.tokens || requests > p.requests || !heads(a[7], tokens, c->kv_heads, c->head_dim, c->dtype, device, &k) ||
      !heads(a[8], tokens, c->kv_heads, c->head_dim, c->dtype, device, &v) || k->strides() != v->strides() ||
      !heads(a[14], tokens, p.q_heads, c->head_dim, c->dtype, device, &out) || !distinct(*out) || table->dim() != 2 || table->size(0) != requests ||
      !ints(a[9], table->numel(), device, false, &p.tables) || !ints(a[10], requests, device, false, &p.context_lens) ||
      !ints(a[11], requests + 1, device, false, &p.starts))
    return status(kUnfit);
  p.mask_words = 0;
  p.mask = nullptr;
  if (a[12] != Py_None) {
    const Tensor* mask = tensor(a[12]);
    const int32_t* bits;
    if (mask == nullptr || mask->dim() != 2 || mask->size(0) < tokens || mask->size(1) * 32 < p.max_new ||
        !ints(a[12], mask->numel(), device, false, &bits))
      return status(kUnfit);
    p.mask = reinterpret_cast<const uint32_t*>(bits);
    p.mask_words = static_cast<uint32_t>(mask->size(1));
  }
  p.lse = nullptr;
  if (a[15] != Py_None) {
    const Tensor* lse = tensor(a[15]);
    if (lse == nullptr || lse->scalar_type() != at::kFloat || lse->dim() != 2 || lse->size(0) != tokens ||
        lse->size(1) != p.q_heads || !lse->is_contiguous() || !lse->is_cuda() || lse->get_device() != device)
      return status(kUnfit);
    p.lse = static_cast<float*>(lse->data_ptr());
  }
  p.requests = static_cast<uint32_t>(requests);
  p.tokens = static_cast<uint32_t>(tokens);
  p.table_stride = static_cast<uint32_t>(table->size(1));
  p.scale = static_cast<float>(PyFloat_AsDouble(a[13]));
  if (PyErr_Occurred() != nullptr) return nullptr;
  p.q = q->const_data_ptr();
  p.k = k->const_data_ptr();
  p.v = v->const_data_ptr();
  p.out = out->data_ptr();
  p.q_token_stride = static_cast<uint64_t>(q->stride(0));
  p.q_head_stride = static_cast<uint64_t>(q->stride(1));
  p.kv_token_stride = static_cast<uint64_t>(k->stride(0));
  p.kv_head_stride = static_cast<uint64_t>(k->stride(1));
  p.out_token_stride = static_cast<uint64_t>(out->stride(0));
  p.out_head_stride = static_cast<uint64_t>(out->stride(1));
  return status(hqb_tree_attention(c, &p, PyLong_AsVoidPtr(a[2]), PyLong_AsUnsignedLongLong(a[3]), stream_of(a[5], device)));
}

// [tokens][cols] of a type, rows that do not overlap; the stride to use (one row has any).
bool rows_of(PyObject* o, int64_t tokens, int64_t cols, int type, int device, const Tensor** t, uint64_t* stride) {
  *t = tensor(o);
  if (*t == nullptr || (*t)->dim() != 2 || (tokens >= 0 && (*t)->size(0) != tokens) || (*t)->size(1) != cols ||
      code((*t)->scalar_type()) != type || !(*t)->is_cuda() || (*t)->get_device() != device || (cols > 1 && (*t)->stride(1) != 1) ||
      ((*t)->size(0) > 1 && (*t)->stride(0) < cols))
    return false;
  *stride = static_cast<uint64_t>((*t)->size(0) > 1 ? (*t)->stride(0) : cols);
  return true;
}

// lora(set address, workspace address, workspace bytes, device, stream, x, ids, base, out)
PyObject* lora(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 9) return status(kUnfit);
  const auto* s = static_cast<const hqb_lora_set*>(PyLong_AsVoidPtr(a[0]));
  const int device = static_cast<int>(PyLong_AsLong(a[3]));
  const OnDevice on(device);
  const Tensor *x, *base = nullptr, *out = tensor(a[8]);
  uint64_t x_stride = 0, base_stride = 0, out_stride = 0;
  const int32_t* ids;
  if (out == nullptr) return status(kUnfit);
  const int kind = code(out->scalar_type());
  if ((kind != s->dtype && kind != HQB_F32) || !rows_of(a[5], -1, static_cast<int64_t>(s->cols), s->dtype, device, &x, &x_stride))
    return status(kUnfit);
  const int64_t tokens = x->size(0);
  if (!ints(a[6], tokens, device, false, &ids) || !rows_of(a[8], tokens, static_cast<int64_t>(s->rows), kind, device, &out, &out_stride) ||
      (a[7] != Py_None && !rows_of(a[7], tokens, static_cast<int64_t>(s->rows), kind, device, &base, &base_stride)))
    return status(kUnfit);
  // base is read ahead of the stores: it is out itself, or elsewhere
  if (base != nullptr && base->data_ptr() != out->data_ptr() && at::get_overlap_status(*base, *out) == at::MemOverlapStatus::Partial)
    return status(kUnfit);
  return status(hqb_lora(s, x->const_data_ptr(), x_stride, ids, static_cast<uint32_t>(tokens),
                         base == nullptr ? nullptr : base->const_data_ptr(), base_stride, out->data_ptr(), kind, out_stride,
                         PyLong_AsVoidPtr(a[1]), PyLong_AsUnsignedLongLong(a[2]), stream_of(a[4], device)));
}

// capture(device, stream) -> hqb_stream_capture's number
PyObject* capture(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 2) return status(kUnfit);
  const OnDevice on(static_cast<int>(PyLong_AsLong(a[0])));
  uint64_t id = 0;
  const int s = hqb_stream_capture(PyLong_AsVoidPtr(a[1]), &id);
  if (s != HQB_OK) return PyErr_Format(PyExc_RuntimeError, "hqb_stream_capture: status %d (%s)", s, hqb_status_string(s));
  return PyLong_FromUnsignedLongLong(id);
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  try {
    PyObject* r = F(self, a, n);
    if (r != nullptr && PyErr_Occurred() != nullptr) {  // a number that is none
      Py_DECREF(r);
      return nullptr;
    }
    return r;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&guarded<F>)), METH_FASTCALL, nullptr};
}

PyMethodDef kMethods[] = {method<page_plan>("page_plan"), method<cache_append>("cache_append"),
                          method<tree_attention>("tree_attention"), method<lora>("lora"), method<capture>("capture"),
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "harpq_b200_bind", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_harpq_b200_bind() { return PyModule_Create(&kModule); }
