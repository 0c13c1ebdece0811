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
// tensors and the numbers of a call.  GradientCalls runs the operators that take a list of tensors
// (neptune_codegen/gradients.py), whose launches hold the tensors' addresses by value.
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/EmptyTensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/library.h>

#include <algorithm>
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

// Whether a tensor's elements are in its storage: not those of a wrapper around other tensors, nor where the storage
// was freed or made shorter behind them (storage.resize_).
bool in_memory(const at::Tensor& t) {
  if (!t.has_storage()) return false;
  if (t.numel() == 0) return true;
  const c10::Storage& storage = t.storage();
  return storage.data() != nullptr && at::detail::computeStorageNbytes(t.sizes(), t.strides(), t.itemsize(),
                                                                       t.storage_offset()) <= storage.nbytes();
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
          t.key_set().has(c10::DispatchKey::Python) || !in_memory(t))
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

// The norm of many tensors and their scaling (csrc/kernels/nep_gradients.h).
class GradientCalls {
 public:
  // tensors of a list by value and of one in device memory, lanes of a workgroup, workgroups of a launch at most
  GradientCalls(int by_value, int most, int lanes, int workgroups)
      : by_value_(by_value), most_(most), lanes_(lanes), workgroups_(workgroups) {
    TORCH_CHECK(by_value > 0 && most >= by_value && lanes > 0 && workgroups > 0, "GradientCalls: bad sizes");
  }

  // A device's kernels: the norm; a part of a long list; sums and scaling of short lists, and of long ones; both
  // at once.
  void add(int device, const std::vector<uint64_t>& kernels) {
    TORCH_CHECK(kernels.size() == 7 && device >= 0, "GradientCalls: expected seven kernels");
    for (uint64_t k : kernels) TORCH_CHECK(k != 0, "GradientCalls: bad kernel");
    kernels_[device] = {kernels[0], kernels[1], kernels[6], {kernels[2], kernels[4]}, {kernels[3], kernels[5]}};
  }
  bool has(int device) const { return kernels_.count(device) != 0; }

  // The tensors' norm (fp32, no dimensions), or None for a list that this does not take.
  py::object norm(const py::handle& tensors) const {
    std::vector<const at::Tensor*> in;
    if (!collect(tensors, in)) return py::none();
    std::vector<Entry> entries;
    entries.reserve(in.size());
    for (const at::Tensor* t : in) push(entries, *t, *t);
    Call call(*this, in[0]->device(), entries);
    at::Tensor out = call.scalar();
    if (call.small()) call.one(out, 0.0f, false, 0);
    else call.norm(call.sums(), out);
    return py::cast(out);
  }

  // `out`: None (in place) or a list.  `given`: None or the norm.  The norm, or None for lists that this does
  // not take.
  py::object clip(const py::handle& tensors, const py::handle& out, const py::handle& given, float max_norm) const {
    std::vector<const at::Tensor*> in, made;
    if (!collect(tensors, in)) return py::none();
    const bool in_place = out.is_none();
    if (!in_place && (!collect(out, made) || made.size() != in.size())) return py::none();
    const std::vector<const at::Tensor*>& to = in_place ? in : made;
    const c10::Device device = in[0]->device();
    std::vector<Entry> entries;
    entries.reserve(in.size());
    int copies = 0;
    for (size_t i = 0; i < in.size(); ++i) {
      const at::Tensor &a = *in[i], &b = *to[i];
      if (b.requires_grad()) return py::none();
      if (!in_place && (b.device() != device || !same_order(a, b) ||
                        (b.scalar_type() != a.scalar_type() && b.scalar_type() != at::kFloat)))
        return py::none();
      push(entries, a, b);
    }
    for (const Entry& e : entries) copies |= e.in != e.out;
    if (!separate(entries)) return py::none();
    at::Tensor norm;
    const bool known = !given.is_none();
    if (known) {
      if (!THPVariable_CheckExact(given.ptr())) return py::none();
      norm = THPVariable_Unpack(given.ptr());
      if (!plain(norm) || norm.device() != device || norm.scalar_type() != at::kFloat || norm.dim() != 0 ||
          inside(norm, entries))
        return py::none();
    }
    Call call(*this, device, entries);
    if (!known) norm = call.scalar();
    if (!known && call.small()) {
      call.one(norm, max_norm, true, copies);
    } else if (!entries.empty()) {
      at::Tensor sums;
      if (!known) sums = call.sums();
      call.scale(sums, norm, known, max_norm, copies);
    }
    for (const at::Tensor* t : to)
      if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
    return py::cast(norm);
  }

 private:
  struct Entry {                                     // TensorEntry of nep_gradients.h
    const void* in;
    void* out;
    uint64_t count;
    uint32_t first, kind;
  };
  static_assert(sizeof(Entry) == 32, "the kernels' layout");
  static constexpr int kPieceLanes = 256;            // as in nep_gradients.h
  static constexpr uint32_t kShort = 8;
  static constexpr uint64_t kSmall = 64 << 10;
  struct Kernels {
    uint64_t norm, list, one, sums[2], scale[2];     // sums and scale of lists by value, and in device memory
  };

  // A launch's arguments.
  struct Image {
    template <class T>
    void put(T value) {
      bytes.resize((bytes.size() + sizeof(T) - 1) / sizeof(T) * sizeof(T));
      const size_t at = bytes.size();
      bytes.resize(at + sizeof(T));
      std::memcpy(bytes.data() + at, &value, sizeof(T));
    }
    std::vector<uint8_t> bytes;
  };

  // One call's lists on its device and stream.
  class Call {
   public:
    Call(const GradientCalls& of, c10::Device device, std::vector<Entry>& entries)
        : of_(of), kernels_(of.kernels_.at(device.index())), guard_(device), entries_(entries),
          options_(at::TensorOptions().device(device)),
          stream_(c10::hip::getCurrentHIPStream(device.index()).stream()) {
      uint64_t total = 0;
      for (const Entry& e : entries_) {
        total += e.count;
        bytes_ += bytes_in(e);
      }
      // two words of a lane (four of 32 bits), up to sixteen where the pieces are many for the workgroups
      while (piece_ < 32 * kPieceLanes * 4 && total / piece_ >= 64ull * of.workgroups_) piece_ *= 2;
      far_ = entries_.size() > static_cast<size_t>(of.by_value_);
      const size_t most = far_ ? of.most_ : of.by_value_;
      for (size_t begin = 0; begin < entries_.size(); begin += most) {
        Part part{begin, std::min(entries_.size(), begin + most), 0};
        uint64_t pieces = 0;
        for (size_t i = part.begin; i < part.end; ++i) {
          entries_[i].first = static_cast<uint32_t>(pieces);
          pieces += (entries_[i].count + piece_ - 1) / piece_;
          TORCH_CHECK_NOT_IMPLEMENTED(pieces < (1ull << 31), "gradients of more than 2^31 pieces of ", piece_,
                                      " elements");
        }
        part.pieces = static_cast<uint32_t>(pieces);
        parts_.push_back(part);
      }
      if (!far_) return;
      // the lists, put together in device memory
      list_ = at::empty({static_cast<int64_t>(entries_.size() * sizeof(Entry))}, options_.dtype(at::kByte));
      for (size_t begin = 0; begin < entries_.size(); begin += of.by_value_) {
        const size_t end = std::min(entries_.size(), begin + of.by_value_);
        Image image;
        by_value(image, begin, end);
        image.put(static_cast<int32_t>(end - begin));
        image.put(device_entries(begin));
        launch(kernels_.list, 1, image);
      }
    }

    // Whether one workgroup does all of it sooner than two launches: 16 KB clipped 5.2 us, 9.5 by two, 78 KB 11.4 and
    // 10.2.  (A norm alone takes 7.2 and 8.7 at 234 KB, but has the order of a clipping's sums, and so its bits.)
    bool small() const { return bytes_ <= kSmall && !far_; }

    void one(at::Tensor& norm, float max_norm, bool scale, int copies) const {
      Image image = head(parts_.empty() ? Part{0, 0, 0} : parts_[0]);
      image.put(norm.data_ptr());
      image.put(max_norm);
      image.put(static_cast<int32_t>(scale));
      image.put(static_cast<int32_t>(copies));
      launch(kernels_.one, 1, image);
    }

    at::Tensor scalar() const { return at::empty({}, options_.dtype(at::kFloat)); }

    // One sum for each workgroup of all launches.
    at::Tensor sums() const {
      int64_t count = 0;
      for (const Part& part : parts_) count += grid(part);
      at::Tensor sums = at::empty({count}, options_.dtype(at::kDouble));
      double* at = static_cast<double*>(sums.data_ptr());
      for (const Part& part : parts_) {
        Image image = head(part);
        image.put(at);
        launch(kernels_.sums[far_], grid(part), image);
        at += grid(part);
      }
      return sums;
    }

    void norm(const at::Tensor& sums, at::Tensor& out) const {
      Image image;
      image.put(sums.data_ptr());
      image.put(static_cast<int32_t>(sums.numel()));
      image.put(out.data_ptr());
      launch(kernels_.norm, 1, image);
    }

    // The first launch writes a norm that is not known.
    void scale(const at::Tensor& sums, at::Tensor& norm, bool known, float max_norm, int copies) const {
      for (const Part& part : parts_) {
        Image image = head(part);
        image.put(known ? nullptr : sums.data_ptr());
        image.put(static_cast<int32_t>(known ? 0 : sums.numel()));
        image.put(known ? norm.data_ptr() : nullptr);
        image.put(!known && part.begin == 0 ? norm.data_ptr() : nullptr);
        image.put(max_norm);
        image.put(static_cast<int32_t>(copies));
        launch(kernels_.scale[far_], copies ? grid(part, kShort) : grid(part), image);
      }
    }

   private:
    struct Part {
      size_t begin, end;                             // entries of one launch
      uint32_t pieces;
    };

    // Workgroups of a launch.  `more`: so many times more where the pieces suffice, since short
    // workgroups keep what is written close together (0.54 GB into fp32 395 us, so 384); not for a scaling in
    // place, which gains nothing (0.54 GB 185 us, by 4096 workgroups 184; 0.1 GB 36 and 36) and often has nothing to
    // do (3.9 us, 6.5).
    uint32_t grid(const Part& part, uint32_t more = 1) const {
      const uint32_t at_once = of_.lanes_ / kPieceLanes, wanted = (part.pieces + at_once - 1) / at_once;
      const uint32_t most = of_.workgroups_;
      return wanted >= more * most ? more * most : std::min(wanted, most);
    }
    const void* device_entries(size_t begin) const {
      return static_cast<const uint8_t*>(list_.data_ptr()) + begin * sizeof(Entry);
    }
    void by_value(Image& image, size_t begin, size_t end) const {
      image.bytes.reserve(of_.by_value_ * sizeof(Entry) + 64);
      image.bytes.resize(of_.by_value_ * sizeof(Entry));
      if (end > begin) std::memcpy(image.bytes.data(), &entries_[begin], (end - begin) * sizeof(Entry));
    }
    // a part's list, its number of entries, its pieces and the elements of a piece
    Image head(const Part& part) const {
      Image image;
      if (far_) image.put(device_entries(part.begin));
      else by_value(image, part.begin, part.end);
      image.put(static_cast<int32_t>(part.end - part.begin));
      image.put(part.pieces);
      image.put(static_cast<int32_t>(piece_));
      return image;
    }
    void launch(uint64_t kernel, uint32_t workgroups, const Image& image) const {
      const int rc = nep_launch_packed(kernel, workgroups, 1, 1, of_.lanes_, 0, stream_, image.bytes.data(),
                                       image.bytes.size());
      if (rc != NEP_OK) throw_hip_error(std::string("launch: ") + nep_last_error());
    }

    const GradientCalls& of_;
    const Kernels& kernels_;
    const c10::DeviceGuard guard_;
    std::vector<Entry>& entries_;
    const at::TensorOptions options_;
    const hipStream_t stream_;
    std::vector<Part> parts_;
    at::Tensor list_;
    uint64_t bytes_ = 0;
    int piece_ = 16 * kPieceLanes;
    bool far_ = false;
  };

  static bool plain(const at::Tensor& t) {
    return t.defined() && t.device().is_cuda() && t.layout() == c10::kStrided && !t.is_neg() && !t.is_conj() &&
           !t.key_set().has(c10::DispatchKey::Python) && in_memory(t);
  }

  // The tensors of a list or tuple that is not empty: of the three types, on one device, without gaps.
  bool collect(const py::handle& list, std::vector<const at::Tensor*>& out) const {
    if (!PyList_CheckExact(list.ptr()) && !PyTuple_CheckExact(list.ptr())) return false;
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(list.ptr());
    if (n == 0) return false;
    out.reserve(n);
    for (Py_ssize_t i = 0; i < n; ++i) {
      PyObject* o = PySequence_Fast_GET_ITEM(list.ptr(), i);
      if (!THPVariable_CheckExact(o)) return false;
      const at::Tensor& t = THPVariable_Unpack(o);
      if (!plain(t) || (i != 0 && t.device() != out[0]->device()) || !t.is_non_overlapping_and_dense())
        return false;
      if (t.scalar_type() != at::kFloat && t.scalar_type() != at::kBFloat16 && t.scalar_type() != at::kHalf)
        return false;
      out.push_back(&t);
    }
    return has(out[0]->get_device());
  }

  // Whether the elements of two tensors without gaps lie in one order.
  static bool same_order(const at::Tensor& a, const at::Tensor& b) {
    if (a.sizes() != b.sizes()) return false;
    for (int64_t d = 0; d < a.dim(); ++d)
      if (a.size(d) != 1 && a.numel() != 0 && a.stride(d) != b.stride(d)) return false;
    return true;
  }

  static void push(std::vector<Entry>& entries, const at::Tensor& in, const at::Tensor& out) {
    if (in.numel() == 0) return;
    const bool wider = in.scalar_type() != at::kFloat && out.scalar_type() == at::kFloat;
    const uint32_t kind = in.scalar_type() == at::kFloat ? 0 : (in.scalar_type() == at::kBFloat16 ? 1 : 2) + 2 * wider;
    entries.push_back({in.data_ptr(), out.data_ptr(), static_cast<uint64_t>(in.numel()), 0, kind});
  }
  static uintptr_t bytes_in(const Entry& e) { return e.count * (e.kind == 0 ? 4 : 2); }
  static uintptr_t bytes_out(const Entry& e) { return e.count * (e.kind == 0 || e.kind > 2 ? 4 : 2); }

  // Whether what is written overlaps nothing else that is written or read, but for a tensor that is written
  // where it is read.
  static bool separate(const std::vector<Entry>& entries) {
    struct Range {
      uintptr_t begin, end;
      bool written;
    };
    std::vector<Range> ranges;
    ranges.reserve(2 * entries.size());
    for (const Entry& e : entries) {
      const auto in = reinterpret_cast<uintptr_t>(e.in), out = reinterpret_cast<uintptr_t>(e.out);
      ranges.push_back({out, out + bytes_out(e), true});
      if (in != out || e.kind > 2) ranges.push_back({in, in + bytes_in(e), false});
    }
    std::sort(ranges.begin(), ranges.end(), [](const Range& a, const Range& b) { return a.begin < b.begin; });
    uintptr_t any = 0, written = 0;                  // ends of the ranges so far
    for (const Range& r : ranges) {
      if (r.begin < (r.written ? any : written)) return false;
      any = std::max(any, r.end);
      if (r.written) written = std::max(written, r.end);
    }
    return true;
  }

  static bool inside(const at::Tensor& t, const std::vector<Entry>& entries) {
    const auto at = reinterpret_cast<uintptr_t>(t.data_ptr());
    for (const Entry& e : entries) {
      const auto begin = reinterpret_cast<uintptr_t>(e.out);
      if (at + 4 > begin && at < begin + bytes_out(e)) return true;
    }
    return false;
  }

  const int by_value_, most_, lanes_, workgroups_;
  std::unordered_map<int, Kernels> kernels_;
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
  m.def("in_memory", &in_memory, py::arg("tensor"));
  py::class_<CallPlan, std::shared_ptr<CallPlan>>(m, "CallPlan")
      .def(py::init<int, const py::tuple&, std::vector<int>, bool, const py::tuple&>(), py::arg("n_inputs"),
           py::arg("buffers"), py::arg("returns"), py::arg("bare"), py::arg("launches"))
      .def("run", &CallPlan::run, py::arg("tensors"));
  py::class_<GradientCalls>(m, "GradientCalls")
      .def(py::init<int, int, int, int>(), py::arg("by_value"), py::arg("most"), py::arg("lanes"),
           py::arg("workgroups"))
      .def("add", &GradientCalls::add, py::arg("device"), py::arg("kernels"))
      .def("has", &GradientCalls::has, py::arg("device"))
      .def("norm", &GradientCalls::norm, py::arg("tensors"))
      .def("clip", &GradientCalls::clip, py::arg("tensors"), py::arg("out"), py::arg("given"), py::arg("max_norm"));
  py::class_<CallTable>(m, "CallTable")
      .def(py::init<>())
      .def("run", &CallTable::run, py::arg("tensors"), py::arg("numbers"))
      .def("keep", &CallTable::keep, py::arg("tensors"), py::arg("numbers"), py::arg("plan"))
      .def("size", &CallTable::size)
      .def("clear", &CallTable::clear);
}
