// The embedding's place in torch's graph, in C++: what ops/embed.py has checked is looked up, and its gradient summed, by the kernels of csrc/embed.cu.
//
// Few tokens cost nothing but host time, and the graph's backward pass runs on a thread of its own where Python takes three times as long as in a loop. 64
// tokens of [32000, 256]: lookup 4.4 us, with a graph 5.7, with its gradient 53; 10.5, 17.9 and 91 from a Python function; 8.2, 9.0 and 59 by the library's.
// Built where there is a compiler for it (_build.load_torch); ops/embed.py does without otherwise. The kernels' entry points are handed over as
// addresses, so that csrc/ stays without torch and this library links to torch alone.
#include <Python.h>
#include <ATen/ATen.h>
#include <ATen/TensorSubclassLikeUtils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/pybind.h>

namespace {

using at::Tensor;
using torch::autograd::variable_list;

// csrc/sx_api.h
typedef long long (*SortedBytes)(long long tokens, long long V);
typedef long long (*Workspace)(long long tokens, long long V, int d, int presorted);
typedef int (*Forward)(const void* ids, int wide, const void* w, long long ldw, void* y, long long tokens, int d, long long V, float scale, int dtype,
                       long long padding, void* sorted, int* status, void* stream);
typedef int (*Backward)(const void* ids, int wide, const void* dy, void* grad, long long ldg, long long tokens, int d, long long V, long long padding,
                        float scale, int add, int dtype, int grad_dtype, const void* sorted, void* work, long long work_bytes, int* status, void* stream);
SortedBytes sorted_bytes;
Workspace workspace;
Forward embed_fwd;
Backward embed_bwd;
constexpr int MOST_DEVICES = 64;
int* status_of[MOST_DEVICES];        // status words, of devices that have been used
PyObject *counter, *name_count, *name_main_grad, *name_written;      // counter: the module whose launch_count counts launches

int code_of(at::ScalarType t) { return t == at::kBFloat16 ? 0 : t == at::kHalf ? 1 : 2; }

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// An attribute of a Python object, or null. The caller has the interpreter.
PyObject* attribute(PyObject* o, PyObject* name) {
  PyObject* v = PyObject_GetAttr(o, name);
  if (!v) PyErr_Clear();
  return v;
}
void count_launch() {
  if (PyObject* n = attribute(counter, name_count)) {
    PyObject* more = PyLong_FromLongLong(PyLong_AsLongLong(n) + 1);
    if (!more || PyObject_SetAttr(counter, name_count, more)) PyErr_Clear();
    Py_XDECREF(more);
    Py_DECREF(n);
  }
}

void sums(const Tensor& grad, const Tensor& ids, const Tensor& dy, double scale, int64_t padding, bool add, const Tensor& order, int* status) {
  const int64_t V = grad.size(0), d = grad.size(1), n = ids.numel();
  const c10::cuda::OptionalCUDAGuard guard(grad.device());
  const long long bytes = workspace(n, V, (int)d, order.defined());
  const Tensor work = at::empty({bytes}, grad.options().dtype(at::kByte));
  const int rc = embed_bwd(ids.const_data_ptr(), ids.scalar_type() == at::kLong, dy.const_data_ptr(), grad.mutable_data_ptr(), grad.stride(0), n, (int)d, V,
                           padding, (float)scale, add, code_of(dy.scalar_type()), code_of(grad.scalar_type()),
                           order.defined() ? order.const_data_ptr() : nullptr, work.mutable_data_ptr(), bytes, status, stream_of(grad));
  TORCH_CHECK(rc == 0, "sx_embed_bwd failed with code ", rc);
}

struct EmbeddingBackward : public torch::autograd::Node {
  torch::autograd::SavedVariable ids;
  Tensor table, order;
  double scale = 1;
  int64_t padding = -1;
  int* status = nullptr;

  std::string name() const override { return "EmbeddingBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    ids.reset_data();
    order.reset();
  }
  variable_list apply(variable_list&& grads) override {
    Tensor i, sorted, dy = grads[0];
    {
      std::lock_guard<std::mutex> lock(mutex_);      // not while the interpreter is waited for
      i = ids.unpack();
      sorted = order;
    }
    if (!dy.defined()) return {Tensor()};
    const int64_t V = table.size(0), d = table.size(1);
    if (at::GradMode::is_enabled() || at::isTensorSubclassLike(dy)) {
      // a graph of this pass, or of a batch of them, is wanted: the same sums by operations that have one
      const Tensor counts = i.ge(0).logical_and(i.lt(V)).logical_and(i.ne(padding));
      const Tensor rows = at::where(counts.unsqueeze(-1), dy.to(at::kFloat) * scale, 0.0).reshape({-1, d});
      return {at::zeros({V, d}, table.options().dtype(at::kFloat)).index_add(0, at::where(counts, i, 0).reshape(-1), rows).to(table.scalar_type())};
    }
    dy = dy.contiguous().resolve_neg();
    Tensor main;
    bool written = false;
    {
      const pybind11::gil_scoped_acquire gil;        // for the table's attributes only: the launches below may have to wait for room
      count_launch();
      PyObject* t = THPVariable_Wrap(table);
      PyObject* g = t ? attribute(t, name_main_grad) : nullptr;
      if (g && THPVariable_Check(g)) {
        main = THPVariable_Unpack(g);
        if ((main.scalar_type() != dy.scalar_type() && main.scalar_type() != at::kFloat) || main.stride(1) != 1) main = Tensor();
      }
      if (main.defined()) {
        PyObject* w = attribute(t, name_written);
        written = w && PyObject_IsTrue(w) == 1;
        Py_XDECREF(w);
        if (PyObject_SetAttr(t, name_written, Py_True)) PyErr_Clear();
      }
      Py_XDECREF(g);
      Py_XDECREF(t);
    }
    if (main.defined()) {
      sums(main, i, dy, scale, padding, written, sorted, status);
      return {Tensor()};
    }
    const Tensor grad = at::empty({V, d}, dy.options());
    sums(grad, i, dy, scale, padding, false, sorted, status);
    return {grad};
  }
};

Tensor looked_up(const Tensor& given, const Tensor& source, double scale, int64_t padding, int* status) {
  const bool train = at::GradMode::is_enabled() && source.requires_grad();
  const Tensor ids = given.contiguous();
  Tensor y, order;
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    const c10::cuda::OptionalCUDAGuard guard(source.device());
    Tensor table = source.resolve_neg();
    const int64_t V = table.size(0), d = table.size(1), n = ids.numel();
    int64_t ldw = table.stride(0);
    if (table.stride(1) != 1 || ldw < d) {
      table = table.contiguous();
      ldw = d;
    }
    c10::SmallVector<int64_t, 6> shape(ids.sizes().begin(), ids.sizes().end());
    shape.push_back(d);
    y = at::empty(shape, table.options());
    const long long bytes = train && d ? sorted_bytes(n, V) : 0;
    if (bytes) order = at::empty({bytes}, table.options().dtype(at::kByte));
    const int rc = embed_fwd(ids.const_data_ptr(), ids.scalar_type() == at::kLong, table.const_data_ptr(), ldw, y.mutable_data_ptr(), n, (int)d, V,
                             (float)scale, code_of(table.scalar_type()), padding, bytes ? order.mutable_data_ptr() : nullptr, status, stream_of(table));
    TORCH_CHECK(rc == 0, "sx_embed_fwd failed with code ", rc);
  }
  if (train) {
    auto node = std::shared_ptr<EmbeddingBackward>(new EmbeddingBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(source));
    node->ids = torch::autograd::SavedVariable(ids, false);
    node->table = source;
    node->order = order;
    node->scale = scale;
    node->padding = padding;
    node->status = status;
    torch::autograd::set_history(y, node);
  }
  return y;
}

// Whether torch has to see no elementary operations on a tensor here (ops/_lib.py: elementary), torch.compile aside.
bool plain(const Tensor& t) { return !at::isTensorSubclassLike(t) && !t._fw_grad(0).defined(); }
bool in_a_transform() {
  return c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode) ||
         c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::Tracer);
}

// (ids, table, scale) -> rows where that is an ordinary call, which is most of them; else None: ops/embed.py looks closer.
PyObject* ordinary(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n == 3 && THPVariable_Check(args[0]) && THPVariable_Check(args[1]) && PyFloat_CheckExact(args[2])) {
    const Tensor& ids = THPVariable_Unpack(args[0]);
    const Tensor& table = THPVariable_Unpack(args[1]);
    const auto type = table.scalar_type(), kind = ids.scalar_type();
    const int dev = table.is_cuda() ? table.get_device() : -1;
    if (dev >= 0 && dev < MOST_DEVICES && status_of[dev] && ids.is_cuda() && ids.get_device() == dev && plain(ids) && plain(table) && !in_a_transform() &&
        table.dim() == 2 && table.size(0) > 0 && (type == at::kBFloat16 || type == at::kHalf || type == at::kFloat) && (kind == at::kLong || kind == at::kInt) &&
        table.layout() == at::kStrided && ids.layout() == at::kStrided) {
      const double scale = PyFloat_AS_DOUBLE(args[2]);
      count_launch();
      Tensor y;
      {
        const pybind11::gil_scoped_release release;
        y = looked_up(ids, table, scale, -1, status_of[dev]);
      }
      return THPVariable_Wrap(std::move(y));
    }
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// (ids, table, scale, padding, address of the status word) -> rows. ids and table have been checked.
PyObject* lookup(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(n == 5 && THPVariable_Check(args[0]) && THPVariable_Check(args[1]), "lookup: two tensors and three numbers");
  TORCH_CHECK(embed_fwd && THPVariable_Unpack(args[0]).is_cuda() && THPVariable_Unpack(args[1]).is_cuda(), "lookup: not bound, or tensors on the CPU");
  const double scale = PyFloat_AsDouble(args[2]);
  const int64_t padding = PyLong_AsLongLong(args[3]);
  int* status = static_cast<int*>(PyLong_AsVoidPtr(args[4]));
  if (PyErr_Occurred()) return nullptr;
  TORCH_CHECK(status, "lookup: no status word");
  const int dev = THPVariable_Unpack(args[1]).get_device();
  if (dev >= 0 && dev < MOST_DEVICES) status_of[dev] = status;
  count_launch();
  Tensor y;
  {
    const pybind11::gil_scoped_release release;
    y = looked_up(THPVariable_Unpack(args[0]), THPVariable_Unpack(args[1]), scale, padding, status);
  }
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// (module that counts launches, addresses of sx_embed_sorted_bytes, sx_embed_bwd_workspace, sx_embed_fwd, sx_embed_bwd)
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(n == 5, "bind: a module and four addresses");
  Py_INCREF(args[0]);
  counter = args[0];
  sorted_bytes = reinterpret_cast<SortedBytes>(PyLong_AsVoidPtr(args[1]));
  workspace = reinterpret_cast<Workspace>(PyLong_AsVoidPtr(args[2]));
  embed_fwd = reinterpret_cast<Forward>(PyLong_AsVoidPtr(args[3]));
  embed_bwd = reinterpret_cast<Backward>(PyLong_AsVoidPtr(args[4]));
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"ordinary", (PyCFunction)(void (*)())ordinary, METH_FASTCALL, nullptr},
    {"lookup", (PyCFunction)(void (*)())lookup, METH_FASTCALL, nullptr},
    {"bind", (PyCFunction)(void (*)())bind, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "libsneppx_torch", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit_libsneppx_torch() {
  name_count = PyUnicode_InternFromString("launch_count");
  name_main_grad = PyUnicode_InternFromString("main_grad");
  name_written = PyUnicode_InternFromString("_main_grad_written");
  return PyModule_Create(&module);
}
