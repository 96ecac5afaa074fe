// Torch-side entry of the paged cache calls: checks the tensors, allocates the
// output and the scratch with torch's caching allocator, fills the argument
// block of include/llmyb.h and makes the call on torch's current stream.
//
// The calls of one decode step take a few microseconds on the GPU; the same
// checks in Python with ctypes took 14-16 us of host time per call, these take
// about 2.  kernels.py holds the documented functions.
#include <Python.h>

#include <cmath>
#include <stdexcept>
#include <string>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../../include/llmyb.h"

namespace {

// raised as ValueError
struct Refused {
  std::string why;
};
[[noreturn]] void refuse(const std::string& why) { throw Refused{why}; }

const at::Tensor* tensor(PyObject* o, const char* name) {
  if (o == Py_None) return nullptr;
  if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a tensor");
  return &THPVariable_Unpack(o);
}

struct Device {
  int index = -1;
  void same(const at::Tensor* t) {
    if (t == nullptr) return;
    if (!t->is_cuda())
      throw std::runtime_error("llmyb kernels take CUDA tensors only (no CPU fallback)");
    if (index < 0) index = t->get_device();
    else if (t->get_device() != index) refuse("paged cache tensors must be on one device");
  }
};

std::string text(const char* name, const char* what) { return std::string(name) + what; }

// [tokens, heads, dim] rows of the cache's type; tokens, heads < 0: any
void* rows(const at::Tensor* t, const char* name, int64_t tokens, int64_t heads, int64_t dim,
           at::ScalarType type, int64_t& token_stride, int64_t& head_stride) {
  if (t == nullptr) refuse(text(name, " is missing"));
  if (t->dim() != 3 || t->scalar_type() != type || t->size(2) != dim ||
      (heads >= 0 && t->size(1) != heads) || (tokens >= 0 && t->size(0) != tokens))
    refuse(text(name, " must be [tokens, heads, head_dim] rows of the cache's type"));
  token_stride = t->stride(0), head_stride = t->stride(1);
  if (t->stride(2) != 1 || (token_stride | head_stride) % 8 != 0 ||
      reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 != 0)
    refuse(text(name, ": contiguous head dimension, 16-byte aligned rows and heads"));
  return t->data_ptr();
}

// what is written has one place per element: by stride, every dimension steps
// over all that the smaller ones span
void apart(const at::Tensor& t, const char* name) {
  int64_t span = 0, last = -1;
  for (int64_t i = 0; i < t.dim(); ++i) {
    int64_t next = -1;  // the smallest stride not yet seen
    for (int64_t d = 0; d < t.dim(); ++d) {
      if (t.size(d) < 2) continue;
      if (t.stride(d) > last && (next < 0 || t.stride(d) < t.stride(next))) next = d;
      for (int64_t e = 0; e < d; ++e)
        if (t.size(e) > 1 && t.stride(e) == t.stride(d)) refuse(text(name, " overlaps itself"));
    }
    if (next < 0) return;
    last = t.stride(next);
    if (last <= span) refuse(text(name, " overlaps itself"));
    span += last * (t.size(next) - 1);
  }
}

template <typename T>
T* vector(const at::Tensor* t, const char* name, at::ScalarType type, int64_t n) {
  if (t == nullptr) return nullptr;
  if (t->dim() != 1 || t->scalar_type() != type || t->size(0) != n || (n > 1 && t->stride(0) != 1))
    refuse(text(name, type == at::kInt ? " must be contiguous int32 [" : " must be contiguous fp32 [") +
           std::to_string(n) + "]");
  return static_cast<T*>(t->data_ptr());
}

int32_t whole(int64_t v, const char* name) {
  if (v < 0 || v > INT32_MAX) refuse(text(name, " is out of range"));
  return static_cast<int32_t>(v);
}

enum Kind { kAppend, kDecode, kPrefill };
const char* const kNames[] = {"llmyb_paged_append", "llmyb_paged_decode", "llmyb_paged_prefill"};

// (kind, q, k, v, k_pages, v_pages, block_table, lengths, cu_q, prefix, slopes,
//  q_norm, k_norm, inv_freq, out, lse, status, scale, softcap, eps, window,
//  interleaved) -> (status code, out)
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  try {
    if (count != 22) refuse("call takes 22 arguments");
    const Kind kind = static_cast<Kind>(PyLong_AsLong(args[0]));
    static const char* const names[] = {"q",      "k",     "v",      "k_pages",  "v_pages",
                                        "block_table", "lengths", "cu_q", "prefix", "slopes",
                                        "q_norm", "k_norm", "inv_freq", "out", "lse"};
    const at::Tensor* t[15];
    Device dev;
    for (int i = 0; i < 15; ++i) dev.same(t[i] = tensor(args[1 + i], names[i]));
    const at::Tensor* const status = tensor(args[16], "status");
    const bool scaled = args[17] != Py_None;
    double scale = scaled ? PyFloat_AsDouble(args[17]) : 1.0;
    const double softcap = PyFloat_AsDouble(args[18]), eps = PyFloat_AsDouble(args[19]);
    const long long window = PyLong_AsLongLong(args[20]);
    const int interleaved = PyObject_IsTrue(args[21]);
    if (PyErr_Occurred()) return nullptr;
    if (!t[0] || !t[3] || !t[4] || !t[5] || !t[6] || !status) refuse("an argument is missing");
    if (dev.index != c10::cuda::current_device())
      refuse("paged cache tensors must be on the current CUDA device");
    const at::Tensor &q = *t[0], &kp = *t[3], &vp = *t[4], &table = *t[5];
    const at::ScalarType type = kp.scalar_type();
    if (kp.dim() != 4 || (type != at::kBFloat16 && type != at::kHalf) || vp.scalar_type() != type ||
        vp.sizes() != kp.sizes() || vp.strides() != kp.strides())
      refuse("k_pages and v_pages must be alike: [pages, kv_heads, page_size, head_dim] bf16 or "
             "fp16 with the same strides");
    llmyb_paged_args a = {};
    a.fp16 = type == at::kHalf;
    a.num_pages = whole(kp.size(0), "the number of pages");
    a.kv_heads = whole(kp.size(1), "kv_heads");
    a.page_size = whole(kp.size(2), "page_size");
    a.head_dim = whole(kp.size(3), "head_dim");
    const int p = a.page_size;
    if ((p != 16 && p != 32 && p != 64 && p != 128 && p != 256) ||
        (a.head_dim != 64 && a.head_dim != 128))
      refuse("pages of 16, 32, 64, 128 or 256 rows and head dimensions 64 or 128 are served");
    a.page_stride = kp.stride(0), a.head_stride = kp.stride(1), a.row_stride = kp.stride(2);
    a.k_pages = kp.data_ptr(), a.v_pages = vp.data_ptr();
    if (kp.stride(3) != 1 || (a.page_stride | a.head_stride | a.row_stride) % 8 != 0 ||
        (reinterpret_cast<uintptr_t>(a.k_pages) | reinterpret_cast<uintptr_t>(a.v_pages)) % 16 != 0)
      refuse("pages: contiguous head dimension, 16-byte aligned pages, heads and rows");
    if (table.dim() != 2 || table.scalar_type() != at::kInt ||
        (table.size(1) > 1 && table.stride(1) != 1))
      refuse("block_table must be int32 [batch, pages per sequence]");
    a.batch = whole(table.size(0), "batch");
    a.table_width = whole(table.size(1), "pages per sequence");
    a.table = static_cast<const int32_t*>(table.data_ptr());
    a.table_stride = table.stride(0);
    a.lengths = vector<int32_t>(t[6], "lengths", at::kInt, a.batch);
    a.q = rows(&q, "q", -1, -1, a.head_dim, type, a.q_token_stride, a.q_head_stride);
    a.n_tokens = whole(q.size(0), "the number of tokens");
    a.q_heads = whole(q.size(1), "the number of heads");
    if (a.kv_heads < 1 || a.q_heads < 1) refuse("at least one head is needed");
    a.cu_q = vector<int32_t>(t[7], "cu_q", at::kInt, static_cast<int64_t>(a.batch) + 1);
    if (!a.cu_q && (kind == kPrefill || a.n_tokens != a.batch))
      refuse(kind == kPrefill ? "cu_q is missing"
                              : "without cu_q there is one token per sequence of block_table");
    int64_t scratch_bytes = 0;
    if (kind == kAppend) {
      apart(kp, "k_pages and v_pages");  // alike
      a.k = rows(t[1], "k", a.n_tokens, a.kv_heads, a.head_dim, type, a.k_token_stride, a.k_head_stride);
      a.v = rows(t[2], "v", a.n_tokens, a.kv_heads, a.head_dim, type, a.v_token_stride, a.v_head_stride);
      const int64_t half = t[12] ? t[12]->numel() : 0;
      if (half % 8 != 0 || 2 * half > a.head_dim)
        refuse("inv_freq must have a multiple of 8 values, at most " + std::to_string(a.head_dim / 2));
      a.rope_half = static_cast<int32_t>(half);
      a.q_norm = vector<float>(t[10], "q_norm", at::kFloat, a.head_dim);
      a.k_norm = vector<float>(t[11], "k_norm", at::kFloat, a.head_dim);
      if ((reinterpret_cast<uintptr_t>(a.q_norm) | reinterpret_cast<uintptr_t>(a.k_norm)) % 16 != 0)
        refuse("q_norm and k_norm must be 16-byte aligned");
      a.inv_freq = vector<float>(t[12], "inv_freq", at::kFloat, half);
      a.interleaved = interleaved;
      a.eps = static_cast<float>(eps);
      if (!(eps >= 0.0)) refuse("eps must be >= 0");
    } else {
      if (a.q_heads % a.kv_heads != 0) refuse("query heads must be a multiple of the kv heads");
      if (!(softcap >= 0.0) || window < 0) refuse("softcap and window must be >= 0 (0: none)");
      if (!scaled) scale = 1.0 / std::sqrt(static_cast<double>(a.head_dim));
      a.scale = static_cast<float>(scale), a.softcap = static_cast<float>(softcap);
      if (!std::isnormal(a.scale) || a.scale < 0.f || !std::isnormal(a.scale * 1.5f))
        refuse("scale must be positive and finite");
      if (softcap > 0.0 && (!std::isnormal(a.softcap * 1.5f) || !std::isnormal(a.scale / a.softcap) ||
                            !std::isnormal(2.f * a.scale / a.softcap)))
        refuse("softcap, or scale / softcap, is beyond what fp32 holds");
      a.window = whole(window, "window");
      a.slopes = vector<float>(t[9], "slopes", at::kFloat, a.q_heads);
      a.prefix = vector<int32_t>(t[8], "prefix", at::kInt, a.batch);
      if (a.prefix && window > 0) refuse("a prefix and a window exclude each other");
      if (const at::Tensor* lse = t[14]) {
        if (lse->scalar_type() != at::kFloat || lse->dim() != 2 || lse->size(0) != a.n_tokens ||
            lse->size(1) != a.q_heads || !lse->is_contiguous())
          refuse("lse must be contiguous fp32 [tokens, heads]");
        a.lse = static_cast<float*>(lse->data_ptr());
      }
      if (kind == kPrefill && a.q_heads > 128 * a.kv_heads)
        refuse("at most 128 query heads per kv head");
      scratch_bytes = kind == kDecode
                          ? llmyb_paged_decode_scratch_bytes(a.q_heads, a.kv_heads, a.head_dim)
                          : llmyb_paged_prefill_scratch_bytes(a.q_heads, a.kv_heads, a.head_dim,
                                                              a.table_width, a.page_size);
    }
    at::Tensor out;
    if (t[13]) {
      out = *t[13];
      apart(out, names[13]);
    } else {
      out = at::empty({a.n_tokens, a.q_heads, a.head_dim}, q.options());
    }
    a.out = rows(&out, "out", a.n_tokens, a.q_heads, a.head_dim, type, a.out_token_stride,
                 a.out_head_stride);
    at::Tensor scratch;
    if (scratch_bytes > 0 && a.n_tokens > 0 && a.batch > 0) {
      scratch = at::empty({scratch_bytes}, q.options().dtype(at::kByte));
      a.scratch = scratch.data_ptr();
    }
    a.dev_status = static_cast<int32_t*>(status->data_ptr());
    void* const stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev.index)).stream();
    const int32_t code = kind == kAppend   ? llmyb_paged_append(&a, stream)
                         : kind == kDecode ? llmyb_paged_decode(&a, stream)
                                           : llmyb_paged_prefill(&a, stream);
    if (code != 0) return Py_BuildValue("(is)", code, kNames[kind]);
    return THPVariable_Wrap(out);
  } catch (const Refused& e) {
    PyErr_SetString(PyExc_ValueError, e.why.c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"call", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(call)), METH_FASTCALL,
     "one paged cache call; kernels.py documents it"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "llmyb_torch", nullptr, -1, methods,
                      nullptr,               nullptr,       nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit_llmyb_torch() {
  return PyModule_Create(&module);
}
