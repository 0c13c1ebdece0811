// _neptune_dispatch: C++ dispatcher kernels for the neptune row-fold operators.
//
// The operators are defined from Python (torch.library.custom_op with a fake impl, as the
// reference does for its Triton ops, neptune_codegen/torch_op.py:16-114), and their Python
// bodies choose a launch configuration, allocate outputs and launch generated HIP kernels.
// Everything those bodies compute is a function of the inputs' dtype, device, sizes, strides
// and 16-byte alignment (no host read of tensor values), so one Python call per such key is
// enough: it runs under a recorder and hands back a *launch plan* -- output/scratch buffer
// shapes plus, per kernel launch, the packed kernarg image with the offsets of its pointer
// arguments.  This file installs, per operator:
//
//   CUDA key          look the key up; on a hit allocate the buffers and replay the launches
//                     on the current stream (no Python, no GIL); on a miss call the Python
//                     body (which validates, launches and records) and keep its plan.
//   AutogradCUDA key  when no input requires grad (or grad mode is off) redispatch below
//                     autograd directly; otherwise hand the call to the operator's original
//                     Python autograd kernel, so gradient behaviour is unchanged.
//
// Calls whose Python body makes a copy of an input, or whose inputs alias one another, leave
// no plan and keep going through Python.
//
// The training operators' direct entry points (neptune_codegen/calls.py) keep their calls here too:
// CallPlan is one call layout's buffers and launches, CallTable finds it again by the layout of the
// tensors and the numbers of a call.
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/library.h>

#include <memory>
#include <mutex>
#include <string>
#include <unordered_map>
#include <vector>

#include "nep_plan.h"

namespace py = pybind11;

namespace {

using nep_plan::Key;
using nep_plan::KeyHash;
using nep_plan::Launch;
using nep_plan::Plan;

// Python callables are held as leaked references: the dispatcher may destroy kernels after
// the interpreter has finalised, when a Py_DECREF would be unsafe.
PyObject* hold(const py::object& fn) {
  PyObject* raw = fn.ptr();
  Py_INCREF(raw);
  return raw;
}

struct Stats {
  int64_t replays = 0, python_calls = 0, plans = 0;
};

// Plans kept per operator; later layouts keep calling the Python body (correct, slower).
constexpr size_t kMaxPlans = 1024;

class PlanKernel final : public c10::OperatorKernel {
 public:
  PlanKernel(int n_inputs, c10::DeviceType device_type, PyObject* body,
             std::shared_ptr<Stats> stats)
      : n_inputs_(n_inputs), device_type_(device_type), body_(body), stats_(std::move(stats)) {}

  void operator()(const c10::OperatorHandle& /*op*/, c10::DispatchKeySet /*ks*/,
                  torch::jit::Stack* stack) {
    auto args = torch::jit::last(*stack, n_inputs_);
    Key key;
    const bool keyed = make_key(args, key);
    std::shared_ptr<const Plan> plan;
    if (keyed) {
      std::lock_guard<std::mutex> guard(mu_);
      auto it = cache_.find(key);
      if (it != cache_.end()) plan = it->second;
    }
    if (plan && plan->replayable) {
      at::Tensor out = replay(*plan, args);
      torch::jit::drop(*stack, n_inputs_);
      torch::jit::push(*stack, std::move(out));
      return;
    }
    at::Tensor out;
    {
      py::gil_scoped_acquire gil;
      bool full;
      {
        std::lock_guard<std::mutex> guard(mu_);
        full = cache_.size() >= kMaxPlans;
      }
      const bool record = keyed && !plan && !full;
      py::tuple call(n_inputs_ + 1);
      call[0] = py::bool_(record);
      for (int i = 0; i < n_inputs_; ++i) call[i + 1] = py::cast(args[i].toTensor());
      py::object result = py::reinterpret_borrow<py::object>(body_)(*call);
      py::tuple pair = result.cast<py::tuple>();
      out = pair[0].cast<at::Tensor>();
      std::shared_ptr<Plan> parsed;
      if (record) parsed = parse_plan(pair[1]);
      std::lock_guard<std::mutex> guard(mu_);
      stats_->python_calls += 1;
      if (parsed) {
        if (parsed->replayable) stats_->plans += 1;
        cache_.emplace(std::move(key), std::move(parsed));
      }
    }
    torch::jit::drop(*stack, n_inputs_);
    torch::jit::push(*stack, std::move(out));
  }

  void clear() {
    std::lock_guard<std::mutex> guard(mu_);
    cache_.clear();
  }

 private:
  bool make_key(c10::ArrayRef<c10::IValue> args, Key& key) const {
    return nep_plan::make_key(args, device_type_, key);
  }

  std::shared_ptr<Plan> parse_plan(const py::handle& spec) const {
    auto plan = std::make_shared<Plan>();
    if (spec.is_none()) return plan;  // known key, Python only
    py::tuple t = spec.cast<py::tuple>();
    for (py::handle b : t[0].cast<py::tuple>()) {
      py::tuple bt = b.cast<py::tuple>();   // (scalar type code, sizes, strides)
      plan->buffers.push_back({bt[1].cast<std::vector<int64_t>>(),
                               bt[2].cast<std::vector<int64_t>>(),
                               static_cast<c10::ScalarType>(bt[0].cast<int>())});
      if (plan->buffers.back().sizes.size() != plan->buffers.back().strides.size())
        return std::make_shared<Plan>();
    }
    for (py::handle l : t[1].cast<py::tuple>()) {
      py::tuple lt = l.cast<py::tuple>();
      Launch launch;
      launch.kernel = lt[0].cast<uint64_t>();
      py::tuple grid = lt[1].cast<py::tuple>();
      for (int d = 0; d < 3; ++d) launch.grid[d] = grid[d].cast<uint32_t>();
      launch.block = lt[2].cast<uint32_t>();
      launch.lds = lt[3].cast<uint32_t>();
      std::string image = lt[4].cast<std::string>();
      launch.image.assign(image.begin(), image.end());
      for (py::handle p : lt[5].cast<py::tuple>()) {
        py::tuple pt = p.cast<py::tuple>();
        launch.patches.emplace_back(pt[0].cast<uint32_t>(), pt[1].cast<int32_t>());
      }
      plan->launches.push_back(std::move(launch));
    }
    // launches need a HIP stream: only device plans may carry them
    plan->replayable = nep_plan::plan_consistent(*plan, n_inputs_) &&
                       (plan->launches.empty() || device_type_ == c10::DeviceType::CUDA);
    return plan;
  }

  at::Tensor replay(const Plan& plan, c10::ArrayRef<c10::IValue> args) {
    at::Tensor out = nep_plan::replay(plan, args);
    std::lock_guard<std::mutex> guard(mu_);
    stats_->replays += 1;
    return out;
  }

  const int n_inputs_;
  const c10::DeviceType device_type_;
  PyObject* const body_;
  std::shared_ptr<Stats> stats_;
  std::mutex mu_;
  std::unordered_map<Key, std::shared_ptr<const Plan>, KeyHash> cache_;
};

class AutogradKernel final : public c10::OperatorKernel {
 public:
  AutogradKernel(int n_inputs, PyObject* grad_body) : n_inputs_(n_inputs), grad_body_(grad_body) {}

  void operator()(const c10::OperatorHandle& op, c10::DispatchKeySet ks,
                  torch::jit::Stack* stack) {
    auto args = torch::jit::last(*stack, n_inputs_);
    bool needs_grad = false;
    if (at::GradMode::is_enabled())
      for (const c10::IValue& arg : args)
        if (arg.isTensor() && arg.toTensor().defined() && arg.toTensor().requires_grad())
          needs_grad = true;
    if (!needs_grad) {
      op.redispatchBoxed(ks & c10::after_autograd_keyset, stack);
      return;
    }
    at::Tensor out;
    {
      py::gil_scoped_acquire gil;
      py::tuple call(n_inputs_);
      for (int i = 0; i < n_inputs_; ++i) call[i] = py::cast(args[i].toTensor());
      out = py::reinterpret_borrow<py::object>(grad_body_)(*call).cast<at::Tensor>();
    }
    torch::jit::drop(*stack, n_inputs_);
    torch::jit::push(*stack, std::move(out));
  }

 private:
  const int n_inputs_;
  PyObject* const grad_body_;
};

struct Installed {
  std::shared_ptr<Stats> stats;
  PlanKernel* kernel;  // owned by the dispatcher
};

std::mutex g_mu;
std::unordered_map<std::string, Installed>& registry() {
  static auto* r = new std::unordered_map<std::string, Installed>();
  return *r;
}

// Library objects are leaked on purpose: their registrations must outlive every caller.
// `backend` is "CUDA" for the operators; "CPU" exists so that the plan cache, the Python
// round trip and the autograd hand-off can be tested without a GPU (plans without launches).
void install(const std::string& qualname, int n_inputs, const py::object& body,
             const py::object& grad_body, const std::string& backend) {
  TORCH_CHECK(n_inputs >= 1, "install: an operator needs at least one tensor input");
  TORCH_CHECK(backend == "CUDA" || backend == "CPU", "install: backend must be CUDA or CPU");
  const bool cuda = backend == "CUDA";
  const auto sep = qualname.find("::");
  TORCH_CHECK(sep != std::string::npos, "install: qualified name expected, got ", qualname);
  std::lock_guard<std::mutex> guard(g_mu);
  TORCH_CHECK(registry().count(qualname) == 0, "install: ", qualname, " is already installed");
  const std::string ns = qualname.substr(0, sep), name = qualname.substr(sep + 2);
  auto stats = std::make_shared<Stats>();
  auto kernel = std::make_unique<PlanKernel>(
      n_inputs, cuda ? c10::DeviceType::CUDA : c10::DeviceType::CPU, hold(body), stats);
  PlanKernel* raw = kernel.get();
  auto* device = new torch::Library(torch::Library::IMPL, ns,
                                    cuda ? c10::DispatchKey::CUDA : c10::DispatchKey::CPU,
                                    __FILE__, __LINE__);
  device->impl(name.c_str(), torch::CppFunction::makeFromBoxedFunctor(std::move(kernel)));
  auto* autograd = new torch::Library(
      torch::Library::IMPL, ns, cuda ? c10::DispatchKey::AutogradCUDA : c10::DispatchKey::AutogradCPU,
      __FILE__, __LINE__);
  autograd->impl(name.c_str(), torch::CppFunction::makeFromBoxedFunctor(
                                   std::make_unique<AutogradKernel>(n_inputs, hold(grad_body))));
  registry().emplace(qualname, Installed{stats, raw});
}

py::dict stats(const std::string& qualname) {
  std::lock_guard<std::mutex> guard(g_mu);
  auto it = registry().find(qualname);
  TORCH_CHECK(it != registry().end(), "stats: ", qualname, " is not installed");
  py::dict d;
  d["replays"] = it->second.stats->replays;
  d["python_calls"] = it->second.stats->python_calls;
  d["plans"] = it->second.stats->plans;
  return d;
}

void clear() {
  std::lock_guard<std::mutex> guard(g_mu);
  for (auto& [name, entry] : registry()) entry.kernel->clear();
}

// The layout key the CUDA kernels compute for these inputs (None when the call has none).
py::object key_of(const std::vector<at::Tensor>& tensors) {
  std::vector<c10::IValue> args(tensors.begin(), tensors.end());
  Key key;
  if (!nep_plan::make_key(args, c10::DeviceType::CUDA, key)) return py::none();
  return py::cast(key);
}

// ---------------------------------------------------------------- direct entry points
// The error that the Python launch path raises (hip.HipError), for entry points that are called from Python.
[[noreturn]] void throw_hip_error(const std::string& message) {
  const py::object type = py::module_::import("neptune_codegen.hip").attr("HipError");
  PyErr_SetString(type.ptr(), message.c_str());
  throw py::error_already_set();
}

// One call layout of an entry point: the buffers it allocates (results first, then scratch) and its
// launches, whose pointer arguments are each an input, or a buffer at a byte offset.
class CallPlan {
 public:
  struct Patch {
    uint32_t offset;        // in the image
    int32_t source;         // input `source`, or buffer -1 - source
    int64_t add;            // bytes
  };
  struct CallLaunch {
    Launch launch;
    std::vector<Patch> patches;
  };

  // buffers: (dtype code, sizes); returns: buffer per result, -1 for None, and whether a single result
  // comes bare; launches: (kernel, grid, block, lds, image, ((offset, source, add), ...))
  CallPlan(int n_inputs, const py::tuple& buffers, std::vector<int> returns, bool bare,
           const py::tuple& launches)
      : n_inputs_(n_inputs), returns_(std::move(returns)), bare_(bare) {
    for (py::handle b : buffers) {
      py::tuple t = b.cast<py::tuple>();
      dtypes_.push_back(static_cast<c10::ScalarType>(t[0].cast<int>()));
      sizes_.push_back(t[1].cast<std::vector<int64_t>>());
    }
    const int n = static_cast<int>(sizes_.size());
    for (int r : returns_) TORCH_CHECK(r >= -1 && r < n, "CallPlan: no such result");
    TORCH_CHECK(!bare_ || (returns_.size() == 1 && returns_[0] >= 0), "CallPlan: one bare result");
    for (py::handle l : launches) {
      py::tuple t = l.cast<py::tuple>();
      CallLaunch c;
      c.launch.kernel = t[0].cast<uint64_t>();
      py::tuple grid = t[1].cast<py::tuple>();
      for (int d = 0; d < 3; ++d) c.launch.grid[d] = grid[d].cast<uint32_t>();
      c.launch.block = t[2].cast<uint32_t>();
      c.launch.lds = t[3].cast<uint32_t>();
      const std::string image = t[4].cast<std::string>();
      c.launch.image.assign(image.begin(), image.end());
      TORCH_CHECK(c.launch.kernel != 0 && image.size() <= nep_plan::kMaxImage, "CallPlan: bad launch");
      for (py::handle p : t[5].cast<py::tuple>()) {
        py::tuple pt = p.cast<py::tuple>();
        Patch patch{pt[0].cast<uint32_t>(), pt[1].cast<int32_t>(), pt[2].cast<int64_t>()};
        TORCH_CHECK(patch.offset + sizeof(void*) <= image.size() && patch.source < n_inputs_ &&
                        -1 - patch.source < n, "CallPlan: bad pointer");
        c.patches.push_back(patch);
      }
      launches_.push_back(std::move(c));
    }
  }

  py::object run(const py::tuple& tensors) const {
    TORCH_CHECK(static_cast<int>(tensors.size()) == n_inputs_, "CallPlan: expected ", n_inputs_, " tensors");
    constexpr int kMostInputs = 16;
    TORCH_CHECK(n_inputs_ <= kMostInputs, "CallPlan: too many tensors");
    char* inputs[kMostInputs];
    const at::Tensor* first = nullptr;
    for (int i = 0; i < n_inputs_; ++i) {
      PyObject* o = PyTuple_GET_ITEM(tensors.ptr(), i);
      inputs[i] = nullptr;
      if (o == Py_None) continue;
      const at::Tensor& t = THPVariable_Unpack(o);
      inputs[i] = static_cast<char*>(t.data_ptr());
      if (first == nullptr) first = &t;
    }
    TORCH_CHECK(first != nullptr, "CallPlan: no tensor");
    const c10::Device device = first->device();
    const c10::DeviceGuard guard(device);
    const at::TensorOptions options = at::TensorOptions().device(device);
    std::vector<at::Tensor> buffers;
    buffers.reserve(sizes_.size());
    for (size_t i = 0; i < sizes_.size(); ++i)
      buffers.push_back(at::empty(sizes_[i], options.dtype(dtypes_[i])));
    if (!launches_.empty()) {
      hipStream_t stream = c10::hip::getCurrentHIPStream(device.index()).stream();
      uint8_t image[nep_plan::kMaxImage];
      for (const CallLaunch& c : launches_) {
        const Launch& l = c.launch;
        std::memcpy(image, l.image.data(), l.image.size());
        for (const Patch& p : c.patches) {
          char* ptr = p.source >= 0 ? inputs[p.source]
                                    : static_cast<char*>(buffers[-1 - p.source].data_ptr()) + p.add;
          std::memcpy(image + p.offset, &ptr, sizeof(ptr));
        }
        const int rc = nep_launch_packed(l.kernel, l.grid[0], l.grid[1], l.grid[2], l.block, l.lds,
                                         stream, image, l.image.size());
        if (rc != NEP_OK) throw_hip_error(std::string("launch: ") + nep_last_error());
      }
    }
    if (bare_) return py::cast(buffers[returns_[0]]);
    py::tuple out(returns_.size());
    for (size_t i = 0; i < returns_.size(); ++i)
      out[i] = returns_[i] < 0 ? py::object(py::none()) : py::cast(buffers[returns_[i]]);
    return out;
  }

 private:
  const int n_inputs_;
  std::vector<c10::ScalarType> dtypes_;
  std::vector<std::vector<int64_t>> sizes_;
  const std::vector<int> returns_;
  const bool bare_;
  std::vector<CallLaunch> launches_;
};

// Plans by (layout of the tensors, numbers): dtype, device, sizes, strides and address mod 16 of plain
// strided device tensors, None for an absent one, and the type and value of each number.  A call with
// anything else among them has no key.
class CallTable {
 public:
  py::object run(const py::tuple& tensors, const py::tuple& numbers) {
    Key key;
    if (!make_key(tensors, numbers, key)) return py::none();
    auto it = plans_.find(key);                      // under the GIL
    if (it == plans_.end()) return py::none();
    const std::shared_ptr<CallPlan> plan = it->second;
    return plan->run(tensors);
  }
  bool keep(const py::tuple& tensors, const py::tuple& numbers, std::shared_ptr<CallPlan> plan) {
    Key key;
    if (!make_key(tensors, numbers, key)) return false;
    if (plans_.size() >= kMostPlans) plans_.clear();
    plans_[std::move(key)] = std::move(plan);
    return true;
  }
  size_t size() const { return plans_.size(); }
  void clear() { plans_.clear(); }

 private:
  static constexpr size_t kMostPlans = 4096;

  static bool make_key(const py::tuple& tensors, const py::tuple& numbers, Key& key) {
    key.reserve(tensors.size() * 14 + numbers.size() * 2);
    for (py::handle h : tensors) {
      PyObject* o = h.ptr();
      if (o == Py_None) {
        key.push_back(-1);
        continue;
      }
      if (!THPVariable_CheckExact(o)) return false;
      const at::Tensor& t = THPVariable_Unpack(o);
      if (!t.defined() || !t.device().is_cuda() || t.layout() != c10::kStrided || t.is_neg() || t.is_conj() ||
          t.key_set().has(c10::DispatchKey::Python))
        return false;
      key.push_back(static_cast<int64_t>(t.scalar_type()));
      key.push_back(t.get_device());
      key.push_back(t.dim());
      for (int64_t s : t.sizes()) key.push_back(s);
      for (int64_t s : t.strides()) key.push_back(s);
      key.push_back(static_cast<int64_t>(reinterpret_cast<uintptr_t>(t.data_ptr()) % 16));
    }
    for (py::handle h : numbers) {
      PyObject* o = h.ptr();
      if (o == Py_None) {
        key.push_back(0);
      } else if (PyBool_Check(o)) {
        key.push_back(o == Py_True ? 2 : 1);
      } else if (PyFloat_CheckExact(o)) {
        const double d = PyFloat_AS_DOUBLE(o);
        int64_t bits;
        std::memcpy(&bits, &d, sizeof(bits));
        key.push_back(3);
        key.push_back(bits);
      } else if (PyLong_CheckExact(o)) {
        int overflow = 0;
        const long long v = PyLong_AsLongLongAndOverflow(o, &overflow);
        if (overflow != 0) return false;
        key.push_back(4);
        key.push_back(v);
      } else {
        return false;
      }
    }
    return true;
  }

  std::unordered_map<Key, std::shared_ptr<CallPlan>, KeyHash> plans_;
};

int64_t dtype_code(const at::Tensor& t) { return static_cast<int64_t>(t.scalar_type()); }

bool installed(const std::string& qualname) {
  std::lock_guard<std::mutex> guard(g_mu);
  return registry().count(qualname) != 0;
}

}  // namespace

PYBIND11_MODULE(_neptune_dispatch, m) {
  m.doc() = "C++ CUDA/AutogradCUDA kernels with launch-plan replay for neptune fold operators";
  m.def("install", &install, py::arg("qualname"), py::arg("n_inputs"), py::arg("body"),
        py::arg("grad_body"), py::arg("backend") = "CUDA");
  m.def("stats", &stats, py::arg("qualname"));
  m.def("clear", &clear);
  m.def("installed", &installed, py::arg("qualname"));
  m.def("key_of", &key_of, py::arg("tensors"));
  m.def("dtype_code", &dtype_code, py::arg("tensor"));
  py::class_<CallPlan, std::shared_ptr<CallPlan>>(m, "CallPlan")
      .def(py::init<int, const py::tuple&, std::vector<int>, bool, const py::tuple&>(), py::arg("n_inputs"),
           py::arg("buffers"), py::arg("returns"), py::arg("bare"), py::arg("launches"))
      .def("run", &CallPlan::run, py::arg("tensors"));
  py::class_<CallTable>(m, "CallTable")
      .def(py::init<>())
      .def("run", &CallTable::run, py::arg("tensors"), py::arg("numbers"))
      .def("keep", &CallTable::keep, py::arg("tensors"), py::arg("numbers"), py::arg("plan"))
      .def("size", &CallTable::size)
      .def("clear", &CallTable::clear);
}
