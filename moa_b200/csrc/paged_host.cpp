// The common case of moa_b200.paged_append and moa_b200.paged_decode on the host, compiled.
//
// A decode step's kernel takes some ten microseconds; checking a dozen tensors and packing their addresses from
// Python takes as long.  The two functions here make the same checks on the tensors' C++ side (1 to 2 us) and
// call the C entry points.  They answer None for everything that is not the common case (a copy to be made, a
// refusal, a capture, another device, a gradient, the first call on a stream): moa_b200/paged.py then does the
// call and raises what there is to raise, so that it alone says what is allowed.
//
// (What the C library is for remains with it: this file adds no kernel and holds no state but the addresses of the
// scratch that paged.py made.)
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <map>
#include <utility>

#include "../../include/moa_b200.h"

namespace {

int (*append_entry)(const moa_paged_append_args*, moa_stream_t) = nullptr;
int (*decode_entry)(const moa_paged_decode_args*, moa_stream_t) = nullptr;
struct Scratch {
  void* at;
  int64_t bytes;
};
std::map<std::pair<int, cudaStream_t>, Scratch> scratch;   // of decode, by device and stream (made by paged.py)
bool known[64];                                            // devices that paged.py has run a call on

const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

// A tensor of the call that can be read where it is: dtype, device, no gradient.
bool fits(const at::Tensor* t, at::ScalarType dtype, int device) {
  return t && t->scalar_type() == dtype && t->is_cuda() && t->get_device() == device &&
         t->layout() == at::kStrided && !(t->requires_grad() && at::GradMode::is_enabled());
}
bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// (a, b, N, D) with rows that the kernels can read; the strides of the first three, a dimension of one counting as zero.
bool rows(const at::Tensor& t, int64_t N, int64_t& a, int64_t& b, int64_t& n) {
  const auto s = t.strides();
  a = s[0];
  b = s[1];
  n = N == 1 ? 0 : s[2];
  return s[3] == 1 && ((a | b | n) & 7) == 0 && aligned(t.data_ptr());
}

bool row_of(const at::Tensor* t, int64_t n, at::ScalarType dtype, int device) {
  return fits(t, dtype, device) && t->dim() == 1 && t->size(0) == n && t->is_contiguous();
}

template <typename A>
bool pool(A& a, const at::Tensor* kp, const at::Tensor* vp, const at::Tensor* table, const at::Tensor* lengths, int64_t B,
          int64_t D, at::ScalarType dtype, int device) {
  if (!fits(kp, dtype, device) || !fits(vp, dtype, device) || kp->dim() != 4 || kp->sizes() != vp->sizes() || kp->size(3) != D)
    return false;
  const auto ks = kp->strides(), vs = vp->strides();
  if (ks[3] != 1 || vs[3] != 1) return false;
  if (!fits(table, at::kInt, device) || table->dim() != 2 || table->size(0) != B ||
      !(table->stride(1) == 1 || table->size(1) == 1) || !row_of(lengths, B, at::kInt, device))
    return false;
  a.k_pages = kp->data_ptr();
  a.v_pages = vp->data_ptr();
  a.page_table = table->const_data_ptr<int32_t>();
  a.lengths = static_cast<int32_t*>(lengths->data_ptr());
  a.kp_page = ks[0]; a.kp_head = ks[1]; a.kp_slot = ks[2];
  a.vp_page = vs[0]; a.vp_head = vs[1]; a.vp_slot = vs[2];
  a.table_stride = table->stride(0);
  a.max_pages = table->size(1);
  a.num_pages = kp->size(0);
  a.page_size = kp->size(2);
  a.KV = kp->size(1);
  a.D = D;
  a.B = B;
  a.dtype = dtype == at::kHalf ? MOA_F16 : MOA_BF16;
  return true;
}

template <typename A>
bool tables(A& a, PyObject* rope, int64_t B, int64_t N, int64_t D, at::ScalarType dtype, int device) {
  if (rope == Py_None) return true;
  if (!PyTuple_Check(rope) || PyTuple_GET_SIZE(rope) != 2) return false;
  const at::Tensor *cos = tensor(PyTuple_GET_ITEM(rope, 0)), *sin = tensor(PyTuple_GET_ITEM(rope, 1));
  if (!cos || !sin) return false;
  const at::ScalarType kind = cos->scalar_type();
  if ((kind != dtype && kind != at::kFloat) || !fits(cos, kind, device) || !fits(sin, kind, device) ||
      cos->sizes() != sin->sizes() || cos->strides() != sin->strides())
    return false;
  const int64_t dim = cos->dim();
  if ((dim != 2 && dim != 3) || cos->size(dim - 1) != D || cos->stride(dim - 1) != 1) return false;
  a.rope_cos = cos->data_ptr();
  a.rope_sin = sin->data_ptr();
  a.rope_f32 = kind == at::kFloat;
  if (dim == 2) {
    if (cos->size(0) <= 0) return false;
    a.rope_sn = cos->stride(0);
    a.rope_rows = cos->size(0);
    return true;
  }
  if ((cos->size(0) != 1 && cos->size(0) != B) || cos->size(1) != N) return false;
  a.rope_sb = cos->size(0) == 1 ? 0 : cos->stride(0);
  a.rope_sn = cos->stride(1);
  return true;
}

// Whether the device is the current one and has been seen by paged.py.
bool ready(int device) { return device >= 0 && device < 64 && known[device] && c10::cuda::current_device() == device; }

// (query, key_pages, value_pages, page_table, lengths, sm_scale, key, value, rope, sink_size, local_size, out, out_dtype,
// advance): the output; None: not the common case; a number: what the C entry point returned.
PyObject* decode(PyObject*, PyObject* const* x, Py_ssize_t n) {
  try {
    if (n != 14) Py_RETURN_NONE;
    const at::Tensor* q = tensor(x[0]);
    if (!q || !q->is_cuda() || q->dim() != 4 || q->size(2) != 1 || x[11] != Py_None || x[12] != Py_None) Py_RETURN_NONE;
    const at::ScalarType dtype = q->scalar_type();
    const int device = q->get_device();
    if ((dtype != at::kHalf && dtype != at::kBFloat16) || !ready(device) || !fits(q, dtype, device)) Py_RETURN_NONE;
    const int64_t B = q->size(0), H = q->size(1), D = q->size(3);
    moa_paged_decode_args a = {};
    if (!pool(a, tensor(x[1]), tensor(x[2]), tensor(x[3]), tensor(x[4]), B, D, dtype, device)) Py_RETURN_NONE;
    int64_t none;
    if (B <= 0 || H <= 0 || a.KV <= 0 || H % a.KV != 0 || !rows(*q, 1, a.q_sb, a.q_sh, none)) Py_RETURN_NONE;
    a.q = q->data_ptr();
    a.H = H;
    a.sm_scale = PyFloat_AsDouble(x[5]);
    const int advance = PyObject_IsTrue(x[13]);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      Py_RETURN_NONE;
    }
    a.advance = advance;
    if (x[6] != Py_None) {
      const at::Tensor *k = tensor(x[6]), *v = tensor(x[7]);
      if (!fits(k, dtype, device) || !fits(v, dtype, device) || k->dim() != 4 || k->sizes() != v->sizes() || k->size(0) != B ||
          k->size(1) != a.KV || k->size(2) != 1 || k->size(3) != D || !rows(*k, 1, a.k_sb, a.k_sh, none) ||
          !rows(*v, 1, a.v_sb, a.v_sh, none) || !tables(a, x[8], B, 1, D, dtype, device))
        Py_RETURN_NONE;
      a.k_new = k->data_ptr();
      a.v_new = v->data_ptr();
    } else if (x[7] != Py_None || x[8] != Py_None || advance) {
      Py_RETURN_NONE;
    }
    if (x[9] != Py_None || x[10] != Py_None) {
      const at::Tensor *sink = tensor(x[9]), *local = tensor(x[10]);
      if (!row_of(sink, a.KV, at::kLong, device) || !row_of(local, a.KV, at::kLong, device)) Py_RETURN_NONE;
      a.sink_size = sink->const_data_ptr<int64_t>();
      a.local_size = local->const_data_ptr<int64_t>();
    }
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(device).stream();
    const auto at_stream = scratch.find({device, stream});
    cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
    if (at_stream == scratch.end()) Py_RETURN_NONE;
    if (cudaStreamIsCapturing(stream, &capturing) != cudaSuccess) {
      (void)cudaGetLastError();
      Py_RETURN_NONE;
    }
    if (capturing != cudaStreamCaptureStatusNone) Py_RETURN_NONE;
    at::Tensor out = at::empty({B, 1, H, D}, q->options().requires_grad(false));
    a.out = out.data_ptr();
    a.o_sb = H * D;
    a.o_sh = D;
    a.workspace = at_stream->second.at;
    a.workspace_bytes = at_stream->second.bytes;
    const int status = decode_entry(&a, stream);
    return status ? PyLong_FromLong(status) : THPVariable_Wrap(std::move(out));
  } catch (...) {                        // whatever it was: paged.py meets it again, and says it
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

// (key, value, key_pages, value_pages, page_table, lengths, counts, rope, query, advance): True without a query, (query, key)
// with one; None and a number as above.
PyObject* append(PyObject*, PyObject* const* x, Py_ssize_t n) {
  try {
    if (n != 10) Py_RETURN_NONE;
    const at::Tensor *k = tensor(x[0]), *v = tensor(x[1]);
    if (!k || !k->is_cuda() || k->dim() != 4) Py_RETURN_NONE;
    const at::ScalarType dtype = k->scalar_type();
    const int device = k->get_device();
    if ((dtype != at::kHalf && dtype != at::kBFloat16) || !ready(device) || !fits(k, dtype, device) || !fits(v, dtype, device) ||
        v->sizes() != k->sizes())
      Py_RETURN_NONE;
    const int64_t B = k->size(0), KV = k->size(1), N = k->size(2), D = k->size(3);
    moa_paged_append_args a = {};
    if (!pool(a, tensor(x[2]), tensor(x[3]), tensor(x[4]), tensor(x[5]), B, D, dtype, device) || a.KV != KV || B <= 0 || KV <= 0 ||
        N <= 0 || !rows(*k, N, a.k_sb, a.k_sh, a.k_sn) || !rows(*v, N, a.v_sb, a.v_sh, a.v_sn) ||
        !tables(a, x[7], B, N, D, dtype, device))
      Py_RETURN_NONE;
    a.k = k->data_ptr();
    a.v = v->data_ptr();
    a.N = N;
    a.H = KV;
    if (x[6] != Py_None) {
      const at::Tensor* counts = tensor(x[6]);
      if (!row_of(counts, B, at::kInt, device)) Py_RETURN_NONE;
      a.counts = counts->const_data_ptr<int32_t>();
    }
    const int advance = PyObject_IsTrue(x[9]);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      Py_RETURN_NONE;
    }
    a.advance = advance;
    at::Tensor q_out, k_out;
    if (x[8] != Py_None) {
      const at::Tensor* q = tensor(x[8]);
      if (!a.rope_cos || !fits(q, dtype, device) || q->dim() != 4 || q->size(0) != B || q->size(1) <= 0 || q->size(2) != N ||
          q->size(3) != D || !rows(*q, N, a.q_sb, a.q_sh, a.q_sn))
        Py_RETURN_NONE;
      a.q = q->data_ptr();
      a.H = q->size(1);
      q_out = at::empty({B, a.H, N, D}, q->options().requires_grad(false));
      k_out = at::empty({B, KV, N, D}, q->options().requires_grad(false));
      a.q_out = q_out.data_ptr();
      a.k_out = k_out.data_ptr();
    }
    const int status = append_entry(&a, c10::cuda::getCurrentCUDAStream(device).stream());
    if (status) return PyLong_FromLong(status);
    if (!a.q) Py_RETURN_TRUE;
    PyObject* both = PyTuple_New(2);
    PyTuple_SET_ITEM(both, 0, THPVariable_Wrap(std::move(q_out)));
    PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(std::move(k_out)));
    return both;
  } catch (...) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

// (address of moa_paged_append, of moa_paged_decode)
PyObject* init(PyObject*, PyObject* args) {
  unsigned long long append_at, decode_at;
  if (!PyArg_ParseTuple(args, "KK", &append_at, &decode_at)) return nullptr;
  append_entry = reinterpret_cast<decltype(append_entry)>(append_at);
  decode_entry = reinterpret_cast<decltype(decode_entry)>(decode_at);
  Py_RETURN_NONE;
}

// (device, stream, address of the scratch or 0, its bytes)
PyObject* seen(PyObject*, PyObject* args) {
  int device;
  unsigned long long stream, at;
  long long bytes;
  if (!PyArg_ParseTuple(args, "iKKL", &device, &stream, &at, &bytes)) return nullptr;
  if (device >= 0 && device < 64) known[device] = append_entry != nullptr;
  if (at) scratch[{device, reinterpret_cast<cudaStream_t>(stream)}] = {reinterpret_cast<void*>(at), bytes};
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"decode", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(decode)), METH_FASTCALL, nullptr},
                         {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(append)), METH_FASTCALL, nullptr},
                         {"init", init, METH_VARARGS, nullptr},
                         {"seen", seen, METH_VARARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// `abi`: of the library whose argument structs are compiled in.
extern "C" PyObject* PyInit__paged_host() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddIntConstant(m, "abi", MOA_ABI_VERSION) != 0) Py_CLEAR(m);
  return m;
}
