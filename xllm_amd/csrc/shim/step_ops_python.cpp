// xllm_amd._step_ops: the functions of step_ops.cpp as a Python module, called by the functions of the same names in
// xllm_amd/ops.py.  The same code is registered with the dispatcher (torch.ops.xllm_ops.*); these calls are a step's
// eager launches, and the dispatcher's way from Python (schema, boxing, keys) was half of their time.
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include "ops_api.h"

namespace {

namespace k = xllm::kernel::mi355;
using torch::Tensor;
using OptTensor = std::optional<Tensor>;

// Positional arguments, unpacked in order.
struct Args {
  PyObject* const* at;
  Args(PyObject* const* args, Py_ssize_t given, Py_ssize_t expected, const char* name) : at(args) {
    TORCH_CHECK_TYPE(given == expected, name, ": ", expected, " arguments expected, ", given, " given");
  }
  Tensor tensor(const char* name) {
    PyObject* x = *at++;
    TORCH_CHECK_TYPE(THPVariable_Check(x), name, " must be a tensor, not ", Py_TYPE(x)->tp_name);
    return THPVariable_Unpack(x);
  }
  OptTensor maybe(const char* name) {
    if (*at == Py_None) {
      ++at;
      return std::nullopt;
    }
    return tensor(name);
  }
  int64_t integer() {
    const long long v = PyLong_AsLongLong(*at++);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
  }
  std::optional<int64_t> maybe_integer() {
    if (*at == Py_None) {
      ++at;
      return std::nullopt;
    }
    return integer();
  }
  double number() {
    const double v = PyFloat_AsDouble(*at++);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
  }
  bool flag() { return *at++ == Py_True; }
  torch::ScalarType dtype() {
    PyObject* x = *at++;
    TORCH_CHECK_TYPE(THPDtype_Check(x), "dtype must be a torch.dtype, not ", Py_TYPE(x)->tp_name);
    return reinterpret_cast<THPDtype*>(x)->scalar_type;
  }
};

PyObject* build_step_tables(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args in(args, n, 8, "build_step_tables");
  const Tensor kv_lens = in.tensor("kv_lens");
  const Tensor new_lens = in.tensor("new_lens");
  const Tensor table = in.tensor("block_table");
  const Tensor free_pages = in.tensor("free_pages");
  const int64_t block_size = in.integer(), budget = in.integer();
  const OptTensor head = in.maybe("free_head");
  PyObject* given = *in.at;   // None, or the seven results
  k::StepTables out;
  if (given == Py_None) {
    out = k::step_tables_memory(kv_lens, budget);
  } else {
    TORCH_CHECK_TYPE(PyTuple_Check(given) && PyTuple_GET_SIZE(given) == 7, "out must be StepTables");
    Args results(reinterpret_cast<PyTupleObject*>(given)->ob_item, 7, 7, "StepTables");
    for (Tensor* t : {&out.block_table, &out.seq_lens, &out.q_cu_seq_lens, &out.position_ids, &out.slot_mapping,
                      &out.new_page_indptr, &out.counters})
      *t = results.tensor("a result");
  }
  {
    pybind11::gil_scoped_release no_gil;
    k::build_step_tables(kv_lens, new_lens, table, free_pages, block_size, budget, head, out);
  }
  if (given != Py_None) Py_RETURN_NONE;
  THPObjectPtr r(PyTuple_New(7));
  if (!r) throw python_error();
  Py_ssize_t i = 0;
  for (const Tensor* t : {&out.block_table, &out.seq_lens, &out.q_cu_seq_lens, &out.position_ids, &out.slot_mapping,
                          &out.new_page_indptr, &out.counters})
    PyTuple_SET_ITEM(r.get(), i++, THPVariable_Wrap(*t));
  return r.release();
  END_HANDLE_TH_ERRORS
}

PyObject* build_cos_sin_cache(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args in(args, n, 7, "build_cos_sin_cache");
  const Tensor inv_freq = in.tensor("inv_freq");
  const OptTensor position_ids = in.maybe("position_ids");
  const int64_t rows = in.integer(), first = in.integer();
  const double factor = in.number();
  const torch::ScalarType dtype = in.dtype();
  const OptTensor given = in.maybe("out");
  Tensor out;
  {
    pybind11::gil_scoped_release no_gil;
    out = k::build_cos_sin_cache(inv_freq, position_ids, rows, first, factor, dtype, given);
  }
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

PyObject* rotary_embedding(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args in(args, n, 10, "rotary_embedding");
  const Tensor position_ids = in.tensor("position_ids");
  const Tensor query = in.tensor("query");
  const OptTensor key = in.maybe("key");
  const Tensor cos_sin = in.tensor("cos_sin_cache");
  const bool interleave = in.flag();
  const int64_t offset = in.integer();
  const std::optional<int64_t> key_offset = in.maybe_integer();
  const bool inverse = in.flag();
  const OptTensor out_query = in.maybe("out_query"), out_key = in.maybe("out_key");
  {
    pybind11::gil_scoped_release no_gil;
    k::rotary_embedding(position_ids, query, key, cos_sin, interleave, offset, key_offset, inverse, out_query, out_key);
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyObject* mla_norm_rope_and_cache(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args in(args, n, 11, "mla_norm_rope_and_cache");
  const Tensor q_pe = in.tensor("q_pe");
  const Tensor kv = in.tensor("kv");
  const Tensor weight = in.tensor("kv_norm_weight");
  const double eps = in.number();
  const Tensor cos_sin = in.tensor("cos_sin_cache");
  const bool interleave = in.flag();
  const Tensor position_ids = in.tensor("position_ids");
  const OptTensor cache = in.maybe("k_cache"), slots = in.maybe("slot_mapping"), out_q = in.maybe("out_q_pe"),
                  out_kv = in.maybe("out_kv");
  {
    pybind11::gil_scoped_release no_gil;
    k::mla_norm_rope_and_cache(q_pe, kv, weight, eps, cos_sin, interleave, position_ids, cache, slots, out_q, out_kv);
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyObject* batch_decode_diff(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args in(args, n, 12, "batch_decode_diff");
  const Tensor query = in.tensor("query");
  const Tensor k_cache = in.tensor("k_cache");
  const Tensor v_cache = in.tensor("v_cache");
  Tensor output = in.tensor("output");
  const Tensor table = in.tensor("block_table");
  const Tensor lens = in.tensor("seq_lens");
  const Tensor lambda = in.tensor("lambda_");
  const double scale = in.number();
  const OptTensor weight = in.maybe("norm_weight");
  const double eps = in.number(), out_scale = in.number();
  const int64_t window = in.integer();
  {
    pybind11::gil_scoped_release no_gil;
    k::batch_decode_diff(query, k_cache, v_cache, output, table, lens, lambda, scale, weight, eps, out_scale, window);
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction fast() {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F));
}
PyMethodDef methods[] = {{"build_step_tables", fast<build_step_tables>(), METH_FASTCALL, nullptr},
                         {"build_cos_sin_cache", fast<build_cos_sin_cache>(), METH_FASTCALL, nullptr},
                         {"rotary_embedding", fast<rotary_embedding>(), METH_FASTCALL, nullptr},
                         {"mla_norm_rope_and_cache", fast<mla_norm_rope_and_cache>(), METH_FASTCALL, nullptr},
                         {"batch_decode_diff", fast<batch_decode_diff>(), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_step_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__step_ops() { return PyModule_Create(&module); }
