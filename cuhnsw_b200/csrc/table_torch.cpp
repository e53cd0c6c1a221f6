// The operators over a table of embeddings for torch tensors: checks of the arguments, results and workspaces from torch's
// allocator, torch's current stream, and one call of the C ABI (include/cuhnsw_b200.h).  Functions of the module
// cuhnsw_b200._table, which cuhnsw_b200/table.py documents and calls with positional arguments.  (Compiled, because the same
// steps in Python take longer than the kernels of a single token: 50 us for a step of a beam search, of which 15 are left.)
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <limits>
#include <memory>
#include <sstream>
#include <stdexcept>
#include <string>
#include <utility>
#include <vector>

#include "../../include/cuhnsw_b200.h"

namespace {

constexpr int64_t kMostIds = (1ll << 31) - 2;
constexpr int64_t kMaxKeep = 256;

template <class... Parts>
[[noreturn]] void refuse(const Parts&... parts) {
  std::ostringstream text;
  (void)std::initializer_list<int>{((text << parts), 0)...};
  throw std::runtime_error(text.str());
}

std::string sizes_text(at::IntArrayRef sizes) {
  std::ostringstream text;
  text << "(";
  for (size_t i = 0; i < sizes.size(); ++i) text << (i ? ", " : "") << sizes[i];
  text << ")";
  return text.str();
}

// -1: no element type of the operators
int type_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return CUHNSW_F32;
    case at::kHalf: return CUHNSW_F16;
    case at::kBFloat16: return CUHNSW_BF16;
    default: return -1;
  }
}

bool is_tensor(PyObject* o) { return THPVariable_Check(o); }

// The tensor with its values in memory: a lazily conjugated or negated one (of torch.conj, torch.imag) as a copy.
at::Tensor unpacked(PyObject* o) {
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_conj() && !t.is_neg()) return t;
  c10::NoGradGuard no_grad;
  return t.resolve_conj().resolve_neg();
}

at::Tensor tensor(PyObject* o, const char* name) {
  if (!is_tensor(o)) refuse(name, " must be a tensor");
  return unpacked(o);
}

bool has_tangent(const at::Tensor& t) { return t._fw_grad(0).defined(); }

// The inputs of an operator without a derivative that one is asked of.  As of torch's own such operators: a tangent is refused
// at the call; a gradient that is recorded is refused where it is asked for, by the results' backward pass.
class Underived {
 public:
  Underived(const char* name, std::initializer_list<PyObject*> inputs) : name_(name) {
    for (PyObject* o : inputs) add(o);
  }
  void add(PyObject* o) {
    if (!is_tensor(o)) return;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (has_tangent(t)) refuse(name_, " has no derivative: a tangent cannot pass through it");
    if (c10::GradMode::is_enabled() && t.requires_grad()) inputs_.push_back(t);
  }
  bool any() const { return !inputs_.empty(); }
  void mark(const at::Tensor& result) const {
    using torch::autograd::NotImplemented;
    if (inputs_.empty() || !torch::autograd::isDifferentiableType(result.scalar_type())) return;
    const std::shared_ptr<NotImplemented> node(new NotImplemented(name_, torch::autograd::collect_next_edges(inputs_)),
                                               torch::autograd::deleteNode);
    torch::autograd::set_history(result, node);
  }

 private:
  const char* name_;
  std::vector<at::Tensor> inputs_;
};

int64_t integer(PyObject* o, const char* name) {
  const long long value = PyLong_AsLongLong(o);
  if (value == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(name, " must be a whole number");
  }
  return value;
}

double number(PyObject* o, const char* name) {
  const double value = PyFloat_AsDouble(o);
  if (value == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(name, " must be a number");
  }
  return value;
}

bool truth(PyObject* o) {
  const int value = PyObject_IsTrue(o);
  if (value < 0) {
    PyErr_Clear();
    refuse("a truth value is expected");
  }
  return value != 0;
}

at::Tensor matrix(PyObject* o, const char* name) {
  const at::Tensor t = tensor(o, name);
  if (!t.is_cuda()) refuse(name, " must be a CUDA tensor");
  if (type_of(t) < 0) refuse(name, " must be float32, float16 or bfloat16, not ", t.scalar_type());
  if (t.dim() != 2) refuse(name, " must have two dimensions, not ", t.dim());
  return t;
}

// `t` with the values of a row next to each other (a copy where they are not)
at::Tensor row_major(const at::Tensor& t) {
  if (t.stride(1) == 1 || t.size(1) == 1) return t;
  c10::NoGradGuard no_grad;
  return t.contiguous();
}
at::Tensor dense(const at::Tensor& t) {
  if (t.is_contiguous()) return t;
  c10::NoGradGuard no_grad;
  return t.contiguous();
}

at::Tensor ids_of(PyObject* o, const at::Device& device) {
  if (!is_tensor(o)) refuse("ids must be an int32 or int64 tensor");
  const at::Tensor ids = unpacked(o);
  if (ids.scalar_type() != at::kInt && ids.scalar_type() != at::kLong) refuse("ids must be an int32 or int64 tensor");
  if (ids.device() != device) refuse("ids are on ", ids.device(), ", the rows on ", device);
  if (ids.numel() > kMostIds) refuse(ids.numel(), " ids are too many");
  return dense(ids);
}

// Whether the memory from a tensor's first value to its last one meets another's.
bool overlap(const at::Tensor& a, const at::Tensor& b) {
  auto range = [](const at::Tensor& t) {
    const uintptr_t begin = reinterpret_cast<uintptr_t>(t.const_data_ptr());
    int64_t last = 0;
    for (int64_t i = 0; i < t.dim(); ++i) last += t.size(i) > 0 ? (t.size(i) - 1) * t.stride(i) : 0;
    return std::pair<uintptr_t, uintptr_t>(begin, t.numel() ? begin + (last + 1) * t.element_size() : begin);
  };
  const auto x = range(a), y = range(b);
  return x.first < y.second && y.first < x.second;
}

at::Tensor make(at::IntArrayRef sizes, at::ScalarType type, const at::Device& device) {
  return at::empty(sizes, at::TensorOptions().dtype(type).device(device));
}

at::Tensor workspace(int64_t bytes, const char* name, const at::Device& device) {
  if (bytes < 0) refuse(name, " failed (", bytes, ")");
  return make({bytes > 0 ? bytes : 1}, at::kByte, device);
}

// One entry point on torch's current stream of `device`, which is the current device meanwhile; other Python threads run.
template <class Call>
void run(const char* name, const at::Device& device, Call call) {
  int rc;
  {
    c10::cuda::CUDAGuard guard(device);
    void* stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
    PyThreadState* state = PyEval_SaveThread();
    rc = call(stream);
    PyEval_RestoreThread(state);
  }
  if (rc != CUHNSW_OK) refuse(name, " failed (", rc, ")");
}

// Python's side of a function: exceptions become RuntimeErrors.
template <PyObject* (*kFunction)(PyObject* const*)>
PyObject* guarded(PyObject*, PyObject* const* args, Py_ssize_t count, Py_ssize_t expected) {
  if (count != expected) {
    PyErr_Format(PyExc_TypeError, "%zd arguments are expected, not %zd", expected, count);
    return nullptr;
  }
  try {
    return kFunction(args);
  } catch (const std::bad_alloc&) {
    PyErr_NoMemory();
  } catch (const c10::OutOfMemoryError& e) {
    PyObject* torch = PyImport_ImportModule("torch");
    PyObject* type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    if (type) PyErr_SetString(type, e.what_without_backtrace());
    Py_XDECREF(type);
    Py_XDECREF(torch);
  } catch (const c10::Error& e) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "unknown failure");
  }
  return nullptr;
}

PyObject* tuple_of(std::initializer_list<at::Tensor> tensors) {
  PyObject* result = PyTuple_New((Py_ssize_t)tensors.size());
  if (!result) throw std::bad_alloc();
  Py_ssize_t i = 0;
  for (const at::Tensor& t : tensors) PyTuple_SET_ITEM(result, i++, THPVariable_Wrap(t));
  return result;
}

// -- rows by number ------------------------------------------------------------------------------------------------------

PyObject* lookup(PyObject* const* args) {  // rows, ids, scale
  const at::Tensor rows = row_major(matrix(args[0], "rows"));
  const at::Device device = rows.device();
  const at::Tensor ids = ids_of(args[1], device);
  const float scale = (float)number(args[2], "scale");
  std::vector<int64_t> sizes = ids.sizes().vec();
  sizes.push_back(rows.size(1));
  const at::Tensor out = make(sizes, rows.scalar_type(), device);
  if (out.numel() > 0)
    run("cuhnsw_lookup_device", device, [&](void* stream) {
      return cuhnsw_lookup_device(rows.const_data_ptr(), rows.stride(0), rows.size(0), rows.size(1), type_of(rows),
                                  ids.const_data_ptr(), ids.scalar_type() == at::kLong, ids.numel(), scale,
                                  out.mutable_data_ptr(), stream);
    });
  return THPVariable_Wrap(out);
}

PyObject* tangent(PyObject* const* args) {  // rows: whether they carry one
  return PyBool_FromLong(is_tensor(args[0]) && has_tangent(THPVariable_Unpack(args[0])));
}

PyObject* lookup_grad(PyObject* const* args) {  // grad, ids, num_rows, scale, out or None, accumulate
  const Underived underived("lookup_grad", {args[0]});
  const at::Tensor given = tensor(args[0], "grad");
  if (!given.is_cuda() || type_of(given) < 0) refuse("grad must be a float32, float16 or bfloat16 CUDA tensor");
  const at::Device device = given.device();
  const at::Tensor ids = ids_of(args[1], device);
  const int64_t rows = integer(args[2], "num_rows"), count = ids.numel();
  const float scale = (float)number(args[3], "scale");
  const bool accumulate = truth(args[5]);
  if (given.dim() != ids.dim() + 1 || given.sizes().slice(0, ids.dim()) != ids.sizes())
    refuse("grad of shape ", sizes_text(given.sizes()), " for ids of shape ", sizes_text(ids.sizes()));
  if (rows < 0 || rows > kMostIds) refuse(rows, " rows are out of range");
  const int64_t dims = given.size(-1);
  at::Tensor grad;
  {
    c10::NoGradGuard no_grad;
    grad = row_major(given.dim() == 2 ? given : given.reshape({count, dims}));
  }
  at::Tensor out;
  if (args[4] == Py_None) {
    if (accumulate) refuse("accumulate needs an out to add to");
    out = make({rows, dims}, grad.scalar_type(), device);
  } else {
    if (is_tensor(args[4])) out = THPVariable_Unpack(args[4]);
    if (!out.defined() || out.device() != device ||
        (out.scalar_type() != grad.scalar_type() && out.scalar_type() != at::kFloat) || out.dim() != 2 ||
        out.size(0) != rows || out.size(1) != dims || !out.is_contiguous())
      refuse("out must be a dense [", rows, ", ", dims, "] tensor of ", grad.scalar_type(), " or float32 on ", device);
    if (out.requires_grad() && c10::GradMode::is_enabled()) refuse("out must not require a gradient");
    if (underived.any()) refuse("out cannot be given for a grad that requires a gradient itself");
    if (out.is_neg()) refuse("out must not be a negated view");
    if (overlap(out, grad) || overlap(out, ids)) refuse("out must not overlap grad or the ids");
    out.unsafeGetTensorImpl()->bump_version();  // whoever keeps it for a backward pass learns that it has changed
  }
  if (out.numel() > 0) {
    const at::Tensor space = workspace(cuhnsw_lookup_grad_workspace(count, rows, dims), "cuhnsw_lookup_grad_workspace", device);
    run("cuhnsw_lookup_grad_device", device, [&](void* stream) {
      return cuhnsw_lookup_grad_device(grad.const_data_ptr(), grad.stride(0), type_of(grad), ids.const_data_ptr(),
                                       ids.scalar_type() == at::kLong, count, rows, dims, scale, out.mutable_data_ptr(),
                                       type_of(out), accumulate, space.mutable_data_ptr(), stream);
    });
  }
  underived.mark(out);
  return THPVariable_Wrap(out);
}

// -- rows in 4 bits ------------------------------------------------------------------------------------------------------

int64_t group_of(PyObject* o) {
  const int64_t group = integer(o, "group");
  if (group != 32 && group != 64 && (group < 128 || group % 128 != 0))
    refuse("group must be 32, 64 or a multiple of 128, not ", group);
  return group;
}

PyObject* pack(PyObject* const* args) {  // rows, group
  const at::Tensor rows = row_major(matrix(args[0], "rows"));
  const int64_t group = group_of(args[1]), n = rows.size(0), d = rows.size(1);
  const at::Device device = rows.device();
  if (d < 1) refuse("rows without dimensions cannot be packed");
  const at::Tensor codes = make({n, 16 * ((d + 31) / 32)}, at::kByte, device);
  const at::Tensor scales = make({n, (d + group - 1) / group}, at::kBFloat16, device);
  run("cuhnsw_pack4_device", device, [&](void* stream) {
    return cuhnsw_pack4_device(rows.const_data_ptr(), rows.stride(0), type_of(rows), n, d, group, codes.mutable_data_ptr(),
                               scales.mutable_data_ptr(), stream);
  });
  return tuple_of({codes, scales});
}

struct Packed {
  at::Tensor codes, scales;
  int64_t n, d, group;
  at::Device device;
};

Packed packed_of(PyObject* const* args) {  // codes, scales, num_dims, group
  const int64_t d = integer(args[2], "num_dims"), group = group_of(args[3]);
  if (d < 1) refuse("num_dims must be at least 1");
  const int64_t width = 16 * ((d + 31) / 32), groups = (d + group - 1) / group;
  at::Tensor codes, scales;
  if (is_tensor(args[0])) codes = unpacked(args[0]);
  if (is_tensor(args[1])) scales = unpacked(args[1]);
  if (!codes.defined() || !codes.is_cuda() || codes.scalar_type() != at::kByte || codes.dim() != 2 ||
      codes.size(1) != width || !codes.is_contiguous() || reinterpret_cast<uintptr_t>(codes.const_data_ptr()) % 16 != 0)
    refuse("codes must be a dense, 16-byte aligned uint8 CUDA tensor [num_rows, ", width, "]");
  if (!scales.defined() || scales.device() != codes.device() || scales.scalar_type() != at::kBFloat16 ||
      scales.dim() != 2 || scales.size(0) != codes.size(0) || scales.size(1) != groups || !scales.is_contiguous())
    refuse("scales must be a dense bfloat16 tensor [", codes.size(0), ", ", groups, "] beside the codes");
  return {codes, scales, codes.size(0), d, group, codes.device()};
}

PyObject* check_packed(PyObject* const* args) {  // codes, scales, num_dims, group
  packed_of(args);
  Py_RETURN_NONE;
}

PyObject* unpack(PyObject* const* args) {  // codes, scales, num_dims, group, dtype
  const Underived underived("PackedRows.unpack", {args[1]});
  const Packed p = packed_of(args);
  if (!THPDtype_Check(args[4])) refuse("dtype must be a torch.dtype");
  const at::ScalarType type = reinterpret_cast<THPDtype*>(args[4])->scalar_type;
  if (type != at::kFloat && type != at::kHalf && type != at::kBFloat16) refuse("cannot unpack to ", type);
  const at::Tensor out = make({p.n, p.d}, type, p.device);
  run("cuhnsw_unpack4_device", p.device, [&](void* stream) {
    return cuhnsw_unpack4_device(p.codes.const_data_ptr(), p.scales.const_data_ptr(), p.n, p.d, p.group,
                                 out.mutable_data_ptr(), type_of(out), stream);
  });
  underived.mark(out);
  return THPVariable_Wrap(out);
}

struct Asked {
  at::Tensor queries, bias;  // no bias: undefined
};

Asked asked_of(const Packed& p, PyObject* queries_given, PyObject* bias_given) {
  const at::Tensor queries = matrix(queries_given, "queries");
  if (queries.device() != p.device) refuse("queries are on ", queries.device(), ", the rows on ", p.device);
  if (queries.size(1) != p.d) refuse("queries have ", queries.size(1), " dimensions, the rows have ", p.d);
  if (queries.size(0) > 1 << 18) refuse(queries.size(0), " queries are too many");
  at::Tensor bias;
  if (bias_given != Py_None) {
    if (is_tensor(bias_given)) bias = unpacked(bias_given);
    if (!bias.defined() || bias.device() != p.device || bias.scalar_type() != at::kFloat || bias.dim() != 1 ||
        bias.size(0) != p.n)
      refuse("bias must be a float32 tensor [", p.n, "] beside the rows");
    bias = dense(bias);
  }
  return {row_major(queries), bias};
}

// Scores of `count` queries from the number `first` on.
at::Tensor scores_of(const Packed& p, const Asked& asked, int64_t first, int64_t count) {
  const at::Tensor out = make({count, p.n}, at::kFloat, p.device);
  const at::Tensor& queries = asked.queries;
  run("cuhnsw_scores4_device", p.device, [&](void* stream) {
    return cuhnsw_scores4_device(p.codes.const_data_ptr(), p.scales.const_data_ptr(), p.n, p.d, p.group,
                                 static_cast<const char*>(queries.const_data_ptr()) +
                                   first * queries.stride(0) * (int64_t)queries.element_size(),
                                 queries.stride(0), type_of(queries), count,
                                 asked.bias.defined() ? asked.bias.const_data_ptr<float>() : nullptr,
                                 out.mutable_data_ptr<float>(), stream);
  });
  return out;
}

PyObject* scores(PyObject* const* args) {  // codes, scales, num_dims, group, queries, bias or None
  const Underived underived("PackedRows.scores", {args[1], args[4], args[5]});
  const Packed p = packed_of(args);
  const Asked asked = asked_of(p, args[4], args[5]);
  const at::Tensor out = scores_of(p, asked, 0, asked.queries.size(0));
  underived.mark(out);
  return THPVariable_Wrap(out);
}

// -- selection -----------------------------------------------------------------------------------------------------------

int64_t keep_of(int64_t keep, const char* name) {
  if (keep < 1 || keep > kMaxKeep) refuse(name, " must be 1 to ", kMaxKeep, ", not ", keep);
  return keep;
}

struct Selected {
  at::Tensor totals, beams, ids, found;
};

// `first`: of the sequences of `out`, the one that the first of these is
void select(const at::Tensor& scores, int64_t seq_stride, int64_t beam_stride, int64_t sequences, int64_t beams,
            int64_t vocabulary, const at::Tensor& totals, int64_t keep, bool log_softmax, bool negate, const Selected& out,
            int64_t first) {
  const at::Device device = scores.device();
  const at::Tensor space =
    workspace(cuhnsw_select_workspace(sequences, beams, vocabulary, (int32_t)keep), "cuhnsw_select_workspace", device);
  run("cuhnsw_select_device", device, [&](void* stream) {
    return cuhnsw_select_device(
      scores.const_data_ptr(), seq_stride, beam_stride, type_of(scores),
      totals.defined() ? totals.const_data_ptr<float>() : nullptr, sequences, beams, vocabulary, (int32_t)keep, log_softmax,
      negate, out.totals.mutable_data_ptr<float>() + first * keep,
      out.beams.defined() ? out.beams.mutable_data_ptr<int32_t>() + first * keep : nullptr,
      out.ids.mutable_data_ptr<int32_t>() + first * keep,
      out.found.defined() ? out.found.mutable_data_ptr<int32_t>() + first : nullptr, space.mutable_data_ptr(), stream);
  });
}

constexpr int64_t kSearchScores = 1ll << 30;  // scores of a search in memory at a time: 4 GB
constexpr int64_t kSearchQueries = 32;        // but so many queries' at least

PyObject* search(PyObject* const* args) {  // codes, scales, num_dims, group, queries, topk, bias or None
  const Underived underived("PackedRows.search", {args[1], args[4], args[6]});
  const Packed p = packed_of(args);
  const int64_t topk = keep_of(integer(args[5], "topk"), "topk");
  const Asked asked = asked_of(p, args[4], args[6]);
  const int64_t count = asked.queries.size(0);
  const Selected out{make({count, topk}, at::kFloat, p.device), {}, make({count, topk}, at::kInt, p.device),
                     make({count}, at::kInt, p.device)};
  if (p.n == 0) {
    out.totals.fill_(std::numeric_limits<float>::infinity());
    out.ids.fill_(-1);
    out.found.zero_();
  } else {
    const int64_t part = std::max(kSearchQueries, kSearchScores / p.n / kSearchQueries * kSearchQueries);
    for (int64_t first = 0; first < count; first += part) {
      const int64_t some = std::min(part, count - first);
      const at::Tensor all = scores_of(p, asked, first, some);
      select(all, p.n, p.n, some, 1, p.n, {}, topk, false, true, out, first);
    }
  }
  underived.mark(out.totals);
  return tuple_of({out.ids, out.totals, out.found});
}

PyObject* select_beams(PyObject* const* args) {  // scores, totals or None, keep or None, log_softmax
  const Underived underived("select_beams", {args[0], args[1]});
  const at::Tensor given = tensor(args[0], "scores");
  if (!given.is_cuda() || type_of(given) < 0) refuse("scores must be a float32, float16 or bfloat16 CUDA tensor");
  if (given.dim() != 3) refuse("scores must be [sequences, beams, vocabulary], not ", given.dim(), "-dimensional");
  const at::Device device = given.device();
  const int64_t sequences = given.size(0), beams = given.size(1), vocabulary = given.size(2);
  const int64_t keep = keep_of(args[2] == Py_None ? beams : integer(args[2], "keep"), "keep");
  const bool log_softmax = truth(args[3]);
  if (beams > 16384) refuse(beams, " beams are too many");
  at::Tensor totals;
  if (args[1] != Py_None) {
    if (is_tensor(args[1])) totals = unpacked(args[1]);
    if (!totals.defined() || totals.device() != device || totals.scalar_type() != at::kFloat || totals.dim() != 2 ||
        totals.size(0) != sequences || totals.size(1) != beams)
      refuse("totals must be a float32 tensor [", sequences, ", ", beams, "] beside the scores");
    totals = dense(totals);
  }
  const at::Tensor scores = given.stride(2) == 1 || vocabulary <= 1 ? given : dense(given);
  const Selected out{make({sequences, keep}, at::kFloat, device), make({sequences, keep}, at::kInt, device),
                     make({sequences, keep}, at::kInt, device), {}};
  if (given.numel() == 0) {
    out.totals.fill_(-std::numeric_limits<float>::infinity());
    out.beams.fill_(-1);
    out.ids.fill_(-1);
  } else {
    select(scores, scores.stride(0), scores.stride(1), sequences, beams, vocabulary, totals, keep, log_softmax, false, out,
           0);
  }
  underived.mark(out.totals);
  return tuple_of({out.totals, out.beams, out.ids});
}

// The rows of a state [sequences, beams, ...] as evenly spaced pieces: how many, values between their beginnings, values of
// each.  False if they are not.
bool pieces_of(const at::Tensor& state, int64_t* segments, int64_t* between, int64_t* each) {
  *segments = *each = 1;
  *between = 0;
  for (int64_t i = state.dim() - 1; i >= 2; --i) {
    const int64_t size = state.size(i), stride = state.stride(i);
    if (size == 1) continue;
    if (*segments == 1 && stride == *each) {
      *each *= size;
    } else if (*segments == 1) {
      *segments = size;
      *between = stride;
    } else if (stride == *segments * *between) {
      *segments *= size;
    } else {
      return false;
    }
  }
  return true;
}

PyObject* pieces(PyObject* const* args) {  // state: (segments, between, each) or None
  int64_t segments, between, each;
  if (!pieces_of(tensor(args[0], "state"), &segments, &between, &each)) Py_RETURN_NONE;
  return Py_BuildValue("LLL", (long long)segments, (long long)between, (long long)each);
}

PyObject* reorder(PyObject* const* args) {  // states, beams
  const bool several = PyList_Check(args[0]) || PyTuple_Check(args[0]);
  if (!several && !is_tensor(args[0])) refuse("states must be a tensor or a list of tensors");
  at::Tensor beams;
  if (is_tensor(args[1])) beams = unpacked(args[1]);
  if (!beams.defined() || !beams.is_cuda() || beams.scalar_type() != at::kInt || beams.dim() != 2)
    refuse("beams must be an int32 CUDA tensor [sequences, keep]");
  beams = dense(beams);
  const at::Device device = beams.device();
  const int64_t sequences = beams.size(0), keep = beams.size(1);
  const Py_ssize_t count = several ? PySequence_Fast_GET_SIZE(args[0]) : 1;
  std::vector<Underived> underived;
  std::vector<at::Tensor> inputs, outs;
  std::vector<cuhnsw_state> states;
  inputs.reserve(count);
  outs.reserve(count);
  states.reserve(count);
  for (Py_ssize_t i = 0; i < count; ++i) {
    PyObject* o = several ? PySequence_Fast_GET_ITEM(args[0], i) : args[0];
    at::Tensor state;
    underived.emplace_back("reorder", std::initializer_list<PyObject*>{o});
    if (is_tensor(o)) state = unpacked(o);
    if (!state.defined() || state.device() != device || state.dim() < 2)
      refuse("a state must be a tensor [sequences, beams, ...] on ", device);
    const at::Tensor& first = i ? inputs[0] : state;
    if (state.size(0) != sequences || state.size(1) != first.size(1))
      refuse("states of shapes ", sizes_text(first.sizes()), " and ", sizes_text(state.sizes()), " for ", sequences,
             " sequences");
    int64_t segments, between, each;
    if (!pieces_of(state, &segments, &between, &each)) {
      state = dense(state);
      pieces_of(state, &segments, &between, &each);
    }
    std::vector<int64_t> sizes = state.sizes().vec();
    sizes[1] = keep;
    at::Tensor out = make(sizes, state.scalar_type(), device);
    const int64_t size = (int64_t)state.element_size();
    states.push_back({state.const_data_ptr(), out.mutable_data_ptr(), state.stride(0) * size, state.stride(1) * size,
                      between * size, each ? segments : 0, each * size});
    inputs.push_back(std::move(state));
    outs.push_back(std::move(out));
  }
  if (count > 0 && sequences > 0 && keep > 0)
    run("cuhnsw_reorder_device", device, [&](void* stream) {
      return cuhnsw_reorder_device(states.data(), (int32_t)count, beams.const_data_ptr<int32_t>(), sequences,
                                   inputs[0].size(1), keep, stream);
    });
  for (Py_ssize_t i = 0; i < count; ++i) underived[i].mark(outs[i]);
  if (!several) return THPVariable_Wrap(outs[0]);
  PyObject* result = PyList_New(count);
  if (!result) throw std::bad_alloc();
  for (Py_ssize_t i = 0; i < count; ++i) PyList_SET_ITEM(result, i, THPVariable_Wrap(outs[i]));
  return result;
}

#define FUNCTION(name, arguments)                                                        \
  {                                                                                      \
    #name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(                   \
             +[](PyObject* self, PyObject* const* args, Py_ssize_t count) -> PyObject* { \
               return guarded<name>(self, args, count, arguments);                       \
             })),                                                                        \
      METH_FASTCALL, nullptr                                                             \
  }

PyMethodDef kMethods[] = {FUNCTION(lookup, 3),  FUNCTION(tangent, 1),      FUNCTION(lookup_grad, 6),  FUNCTION(pack, 2),
                          FUNCTION(check_packed, 4), FUNCTION(unpack, 5),  FUNCTION(scores, 6),       FUNCTION(search, 7),
                          FUNCTION(select_beams, 4), FUNCTION(pieces, 1),  FUNCTION(reorder, 2),      {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_table", "The operators over a table of embeddings for torch tensors.",
                       -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__table(void) { return PyModule_Create(&kModule); }
