// tensors.cpp -- the tensor-level calls of sampling and the experts' operators as a Python module.
//
// A small call on the GPU takes a few microseconds, and checking tensors, allocating outputs and
// crossing ctypes from Python takes about eight; here the same work takes about two.  Every function
// checks its arguments (ValueError), allocates its outputs, and calls the C ABI of
// include/batch_topk_b200.h on the current stream of its tensors' device (BatchTopkError).  The
// gradients of route, dispatch and combine are autograd nodes of this module.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/core/Allocator.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <string>
#include <utility>

#include "../../include/batch_topk_b200.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Refused : std::invalid_argument {  // a ValueError
  using std::invalid_argument::invalid_argument;
};
struct Failed : std::runtime_error {  // a BatchTopkError
  int code;
  const char* name;
  Failed(int c, const char* n)
      : std::runtime_error(std::string(n) + ": " + bt_error_string(c)), code(c), name(n) {}
};

std::string text_of(const char* s) { return s; }
std::string text_of(const at::Device& d) { return d.str(); }
std::string text_of(double v) {
  char t[32];
  std::snprintf(t, sizeof(t), "%g", v);
  return t;
}
template <class I, class = std::enable_if_t<std::is_integral_v<I>>>
std::string text_of(I v) {
  return std::to_string(v);
}

template <class... A>
[[noreturn]] void refuse(const A&... parts) {
  throw Refused((std::string() + ... + text_of(parts)));
}

void check(int code, const char* what) {
  if (code != 0) throw Failed(code, what);
}

// A dual tensor's tangent would be lost.
void no_tangent(const at::Tensor& t) {
  TORCH_CHECK(!t._fw_grad(0).defined() ||
                  !c10::AutogradState::get_tls_state().get_fw_grad_mode(),
              "route, dispatch and combine have no forward-mode derivatives");
}
void first_order(const at::Tensor& grad) {
  no_tangent(grad);
  TORCH_CHECK(!(at::GradMode::is_enabled() && grad.requires_grad()),
              "route, dispatch and combine have first-order gradients only");
}
bool wants_grad(const at::Tensor& t) {
  no_tangent(t);
  return t.requires_grad() && at::GradMode::is_enabled();
}

// A gradient under create_graph, which depends on `source` beside the upstream gradient: the same
// values with a node that refuses to be differentiated, so that no term is dropped on the way to
// source.
struct OnceNode : torch::autograd::Function<OnceNode> {
  static at::Tensor forward(AutogradContext*, const at::Tensor& gradient, const at::Tensor&) {
    return gradient.alias();
  }
  static variable_list backward(AutogradContext*, const variable_list&) {
    TORCH_CHECK(false, "route, dispatch and combine have first-order gradients only");
  }
};
at::Tensor once(const at::Tensor& gradient, const at::Tensor& source) {
  const bool graph = gradient.defined() && at::GradMode::is_enabled() && source.requires_grad();
  return graph ? OnceNode::apply(gradient, source) : gradient;
}

PyObject* raise(const Refused& r) {
  PyErr_SetString(PyExc_ValueError, r.what());
  return nullptr;
}

PyObject* raise(const Failed& f) {
  PyObject* package = PyImport_ImportModule("batch_topk_b200");
  PyObject* type = package ? PyObject_GetAttrString(package, "BatchTopkError") : nullptr;
  PyObject* error = type ? PyObject_CallFunction(type, "is", f.code, f.name) : nullptr;
  if (error) PyErr_SetObject(type, error);
  Py_XDECREF(error);
  Py_XDECREF(type);
  Py_XDECREF(package);
  return nullptr;
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse(name, " must be a tensor");
  return THPVariable_Unpack(o);
}

int elem_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kHalf: return BT_DTYPE_F16;
    case at::kBFloat16: return BT_DTYPE_BF16;
    case at::kFloat: return BT_DTYPE_F32;
    default: return -1;
  }
}

// The rows of a 2-D tensor of values: its element type, and itself or a copy with adjacent values.
int rows_of(const at::Tensor& t, const char* name) {
  const int elem = elem_of(t);
  if (elem < 0 || t.dim() != 2 || !t.is_cuda()) {
    refuse(name, " must be a 2-D float16, bfloat16 or float32 CUDA tensor");
  }
  return elem;
}
at::Tensor row_major(const at::Tensor& t) {
  return t.stride(1) == 1 || t.size(1) <= 1 ? t : t.contiguous();
}

// The library launches on the current device and the given stream.
struct Place {
  c10::cuda::CUDAGuard guard;
  void* stream;
  explicit Place(const at::Tensor& t)
      : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.get_device()).stream()) {}
};

at::Tensor empty(at::IntArrayRef size, const at::Tensor& like, at::ScalarType type) {
  return at::empty(size, like.options().dtype(type).requires_grad(false));
}

int small(int64_t v, const char* name) {
  if (v > 0x7FFFFFFF) refuse(name, " is too large: ", v);
  return static_cast<int>(v);
}

PyObject* pack(const at::Tensor& a, const at::Tensor& b) {
  PyObject* t = PyTuple_New(2);
  if (!t) return nullptr;
  PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(a));
  PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(b));
  return t;
}

long long integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw python_error();
  return v != 0;
}

// ---- sampling --------------------------------------------------------------------------------

// One setting: a number of its range for the batch, or a tensor of its type with one for each row.
struct Setting {
  double value = 0.0;
  at::Tensor rows;
  const void* data() const { return rows.defined() ? rows.data_ptr() : nullptr; }
};

Setting setting(PyObject* o, const char* name, const at::Tensor& logits, at::ScalarType type,
                double lo, double hi) {
  Setting s;
  if (THPVariable_Check(o)) {
    const at::Tensor& t = THPVariable_Unpack(o);
    if (t.scalar_type() != type || t.dim() != 1 || t.size(0) != logits.size(0) ||
        t.device() != logits.device()) {
      refuse(name, " must be a number or a ", type == at::kInt ? "int32" : "float32", " tensor [",
             logits.size(0), "] on ", logits.device());
    }
    s.rows = t.contiguous();
    return s;
  }
  s.value = type == at::kInt ? static_cast<double>(integer(o)) : number(o);
  if (!(s.value >= lo && s.value <= hi)) {
    refuse(name, " must lie in [", lo, ", ", hi, "], got ", s.value);
  }
  return s;
}

// sample(logits, noise, temperature, top_k, top_p, min_p, out or None)
PyObject* sample(PyObject* const* a) {
  const at::Tensor& given = tensor(a[0], "logits");
  const int elem = rows_of(given, "logits");
  const at::Tensor& given_noise = tensor(a[1], "noise");
  const int64_t rows = given.size(0), vocab = given.size(1);
  if (given_noise.scalar_type() != at::kFloat || given_noise.sizes() != given.sizes() ||
      given_noise.device() != given.device()) {
    refuse("noise must be a float32 tensor of the logits' shape on their device");
  }
  if (vocab < 1 || vocab > BT_MAX_SEG_LEN) {
    refuse("vocab must lie in [1, ", BT_MAX_SEG_LEN, "], got ", vocab);
  }
  const double inf = std::numeric_limits<double>::infinity();
  const Setting t = setting(a[2], "temperature", given, at::kFloat, 0.0, inf);
  const Setting k = setting(a[3], "top_k", given, at::kInt, 0.0, 2147483647.0);
  const Setting p = setting(a[4], "top_p", given, at::kFloat, 0.0, 1.0);
  const Setting m = setting(a[5], "min_p", given, at::kFloat, 0.0, 1.0);
  const Place place(given);
  at::Tensor tokens, logprobs;
  if (a[6] == Py_None) {
    tokens = empty({rows}, given, at::kInt);
    logprobs = empty({rows}, given, at::kFloat);
  } else {
    if (!PyTuple_Check(a[6]) || PyTuple_GET_SIZE(a[6]) != 2) refuse("out must be a pair of tensors");
    tokens = tensor(PyTuple_GET_ITEM(a[6], 0), "out");
    logprobs = tensor(PyTuple_GET_ITEM(a[6], 1), "out");
    for (const at::Tensor* o : {&tokens, &logprobs}) {
      if (o->scalar_type() != (o == &tokens ? at::kInt : at::kFloat) || o->dim() != 1 ||
          o->size(0) != rows || o->device() != given.device() || !o->is_contiguous()) {
        refuse("out must be contiguous int32 and float32 tensors [", rows, "] on ", given.device());
      }
    }
  }
  if (rows > 0) {
    const at::Tensor logits = row_major(given), noise = row_major(given_noise);
    check(bt_sample(logits.data_ptr(), elem, small(rows, "the number of rows"),
                    static_cast<int>(vocab), logits.stride(0), noise.data_ptr<float>(),
                    noise.stride(0), static_cast<float>(t.value),
                    static_cast<const float*>(t.data()), static_cast<int>(k.value),
                    static_cast<const int*>(k.data()), static_cast<float>(p.value),
                    static_cast<const float*>(p.data()), static_cast<float>(m.value),
                    static_cast<const float*>(m.data()), tokens.data_ptr<int>(),
                    logprobs.data_ptr<float>(), place.stream),
          "sample");
  }
  return pack(tokens, logprobs);
}

// ---- routing ---------------------------------------------------------------------------------

int score_of(PyObject* o) {
  const char* name = PyUnicode_Check(o) ? PyUnicode_AsUTF8(o) : "";
  if (!name) throw python_error();  // a UnicodeEncodeError, which is a ValueError
  if (std::string("softmax") == name) return BT_SCORE_SOFTMAX;
  if (std::string("sigmoid") == name) return BT_SCORE_SIGMOID;
  refuse("score must be \"softmax\" or \"sigmoid\", got \"", name, "\"");
}

struct RouteArgs {
  int elem, k, score, groups, topk_groups, renormalize;
  float scale;
  at::Tensor bias;  // or none; not an argument of the node, as it has no gradient
};

std::pair<at::Tensor, at::Tensor> route_forward(const at::Tensor& given, const RouteArgs& a) {
  const Place place(given);
  at::Tensor weights = empty({given.size(0), a.k}, given, at::kFloat);
  at::Tensor chosen = empty({given.size(0), a.k}, given, at::kInt);
  if (given.size(0) > 0) {
    const at::Tensor logits = row_major(given);
    check(bt_route(logits.data_ptr(), a.elem, static_cast<int>(logits.size(0)),
                   static_cast<int>(logits.size(1)), logits.stride(0), a.k, a.score,
                   a.bias.defined() ? a.bias.data_ptr<float>() : nullptr, a.groups, a.topk_groups,
                   a.renormalize, a.scale, weights.data_ptr<float>(), chosen.data_ptr<int>(),
                   place.stream),
          "route");
  }
  return {weights, chosen};
}

struct RouteNode : torch::autograd::Function<RouteNode> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& logits,
                               const RouteArgs& a) {
    auto [weights, chosen] = route_forward(logits, a);
    ctx->save_for_backward({logits, chosen});
    ctx->saved_data["score"] = a.score;
    ctx->saved_data["renormalize"] = a.renormalize;
    ctx->saved_data["scale"] = static_cast<double>(a.scale);
    ctx->mark_non_differentiable({chosen});
    ctx->set_materialize_grads(false);
    return {weights, chosen};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    if (!grads[0].defined()) return {at::Tensor(), at::Tensor()};
    first_order(grads[0]);
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor logits = row_major(saved[0]), &chosen = saved[1];
    const at::Tensor grad = grads[0].to(at::kFloat).contiguous();
    const Place place(logits);
    at::Tensor out = empty({logits.size(0), logits.size(1)}, logits, logits.scalar_type());
    if (logits.size(0) > 0) {
      check(bt_route_backward(logits.data_ptr(), elem_of(logits), static_cast<int>(logits.size(0)),
                              static_cast<int>(logits.size(1)), logits.stride(0),
                              static_cast<int>(chosen.size(1)),
                              static_cast<int>(ctx->saved_data["score"].toInt()),
                              static_cast<int>(ctx->saved_data["renormalize"].toInt()),
                              static_cast<float>(ctx->saved_data["scale"].toDouble()),
                              chosen.data_ptr<int>(), grad.data_ptr<float>(), out.data_ptr(),
                              place.stream),
            "route backward");
    }
    return {once(out, saved[0]), at::Tensor()};
  }
};

// route(logits, k, score, bias or None, groups, topk_groups, renormalize, scale)
PyObject* route(PyObject* const* a) {
  const at::Tensor& given = tensor(a[0], "logits");
  const int elem = rows_of(given, "logits");
  const int64_t tokens = given.size(0), experts = given.size(1);
  const long long k = integer(a[1]), groups = integer(a[4]), topk_groups = integer(a[5]);
  const int score = score_of(a[2]);
  if (experts < 1 || experts > BT_MAX_EXPERTS) {
    refuse("1 to ", BT_MAX_EXPERTS, " experts are supported, got ", experts);
  }
  if (groups < 1 || groups > 32 || experts % groups != 0 || topk_groups < 1 ||
      topk_groups > groups) {
    refuse("groups=", groups, ", topk_groups=", topk_groups, ": groups (at most 32) must divide ",
           experts, " experts, topk_groups must lie in [1, groups]");
  }
  if (k < 1 || k > BT_MAX_EXPERTS_PER_TOKEN || k > experts / groups * topk_groups) {
    refuse("k=", k, ": 1 to min(", BT_MAX_EXPERTS_PER_TOKEN,
           ", experts that stay) are supported");
  }
  at::Tensor bias;
  if (a[3] != Py_None) {
    bias = tensor(a[3], "bias");
    if (bias.scalar_type() != at::kFloat || bias.dim() != 1 || bias.size(0) != experts ||
        bias.device() != given.device()) {
      refuse("bias must be a float32 tensor [", experts, "] on ", given.device());
    }
    bias = bias.contiguous();
  }
  const RouteArgs args{elem, static_cast<int>(k), score, static_cast<int>(groups),
                       static_cast<int>(topk_groups), truth(a[6]),
                       static_cast<float>(number(a[7])), bias};
  small(tokens, "the number of tokens");
  if (wants_grad(given)) {
    const variable_list out = RouteNode::apply(given, args);
    return pack(out[0], out[1]);
  }
  const auto [weights, chosen] = route_forward(given, args);
  return pack(weights, chosen);
}

// ---- the experts' rows -------------------------------------------------------------------------

// expert_order(experts, num_experts)
PyObject* expert_order(PyObject* const* a) {
  const at::Tensor& given = tensor(a[0], "experts");
  const long long num = integer(a[1]);
  if (given.scalar_type() != at::kInt || given.dim() != 2 || !given.is_cuda()) {
    refuse("experts must be a 2-D int32 CUDA tensor");
  }
  if (num < 1 || num > BT_MAX_EXPERTS) {
    refuse("1 to ", BT_MAX_EXPERTS, " experts are supported, got ", num);
  }
  const int64_t n = given.numel();
  if (n > BT_MAX_ASSIGNMENTS) {
    refuse("at most ", BT_MAX_ASSIGNMENTS, " assignments are supported, got ", n);
  }
  const Place place(given);
  at::Tensor offsets = empty({num + 1}, given, at::kInt);
  at::Tensor order = empty({n}, given, at::kInt);
  at::Tensor position = empty({given.size(0), given.size(1)}, given, at::kInt);
  if (n == 0) {
    offsets.zero_();
  } else {
    const at::Tensor experts = given.contiguous();
    const size_t bytes = bt_expert_order_workspace_size(static_cast<int>(n), static_cast<int>(num));
    // The call's own: it goes back to the allocator in the stream's order, and what a CUDA graph
    // captured belongs to that graph.
    const c10::DataPtr scratch = c10::GetAllocator(at::kCUDA)->allocate(bytes);
    check(bt_expert_order(experts.data_ptr<int>(), static_cast<int>(n), static_cast<int>(num),
                          offsets.data_ptr<int>(), order.data_ptr<int>(), position.data_ptr<int>(),
                          scratch.get(), bytes, place.stream),
          "expert_order");
  }
  PyObject* t = PyTuple_New(3);
  if (!t) return nullptr;
  PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(offsets));
  PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(order));
  PyTuple_SET_ITEM(t, 2, THPVariable_Wrap(position));
  return t;
}

// A plan's three tensors, on the device of `like`.
struct Plan {
  at::Tensor offsets, order, position;
  int tokens, k;
};

Plan plan_of(PyObject* o, const at::Tensor& like) {
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 3) refuse("plan must be an ExpertOrder");
  const char* names[3] = {"offsets", "order", "position"};
  for (int i = 0; i < 3; ++i) {
    const at::Tensor& t = tensor(PyTuple_GET_ITEM(o, i), names[i]);
    const int dim = i == 2 ? 2 : 1;
    if (t.scalar_type() != at::kInt || t.dim() != dim || t.device() != like.device() ||
        !t.is_contiguous()) {
      refuse("plan.", names[i], " must be a contiguous ", dim, "-D int32 tensor on ",
             like.device());
    }
  }
  const at::Tensor& offsets = THPVariable_Unpack(PyTuple_GET_ITEM(o, 0));
  const at::Tensor& order = THPVariable_Unpack(PyTuple_GET_ITEM(o, 1));
  const at::Tensor& position = THPVariable_Unpack(PyTuple_GET_ITEM(o, 2));
  const int64_t n = position.size(0), k = position.size(1);
  if (order.numel() != n * k || offsets.numel() < 2) {
    refuse("plan.order must hold one place for each entry of plan.position");
  }
  if (k < 1 || k > BT_MAX_EXPERTS_PER_TOKEN || n * k > BT_MAX_ASSIGNMENTS) {
    refuse("1 to ", BT_MAX_EXPERTS_PER_TOKEN, " experts a token and at most ", BT_MAX_ASSIGNMENTS,
           " assignments are supported, got ", n, " x ", k);
  }
  return Plan{offsets, order, position, static_cast<int>(n), static_cast<int>(k)};
}

at::Tensor dispatch_forward(const at::Tensor& given, const Plan& plan) {
  const Place place(given);
  at::Tensor rows = empty({static_cast<int64_t>(plan.tokens) * plan.k, given.size(1)}, given,
                          given.scalar_type());
  if (rows.numel() > 0) {
    const at::Tensor x = row_major(given);
    check(bt_dispatch(x.data_ptr(), elem_of(x), plan.tokens, plan.k, static_cast<int>(x.size(1)),
                      x.stride(0), plan.order.data_ptr<int>(), rows.data_ptr(), place.stream),
          "dispatch");
  }
  return rows;
}

// weights undefined: weights of 1
at::Tensor combine_forward(const at::Tensor& given, const at::Tensor& position,
                           const at::Tensor& weights) {
  const Place place(given);
  at::Tensor y = empty({position.size(0), given.size(1)}, given, given.scalar_type());
  if (y.numel() > 0) {
    const at::Tensor rows = given.contiguous();
    check(bt_combine(rows.data_ptr(), elem_of(rows), static_cast<int>(position.size(0)),
                     static_cast<int>(position.size(1)), static_cast<int>(rows.size(1)),
                     position.data_ptr<int>(),
                     weights.defined() ? weights.data_ptr<float>() : nullptr, y.data_ptr(),
                     place.stream),
          "combine");
  }
  return y;
}

struct DispatchNode : torch::autograd::Function<DispatchNode> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const Plan& plan) {
    ctx->save_for_backward({plan.position});
    return dispatch_forward(x, plan);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    first_order(grads[0]);
    return {combine_forward(grads[0], ctx->get_saved_variables()[0], at::Tensor()), at::Tensor()};
  }
};

struct CombineNode : torch::autograd::Function<CombineNode> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& rows,
                            const at::Tensor& weights, const Plan& plan) {
    ctx->save_for_backward({rows, weights, plan.offsets, plan.position});
    return combine_forward(rows, plan.position, weights.contiguous());
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    first_order(grads[0]);
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor rows = saved[0].contiguous(), weights = saved[1].contiguous();
    const at::Tensor &offsets = saved[2], &position = saved[3], grad = row_major(grads[0]);
    const Place place(rows);
    at::Tensor d_rows, d_weights;
    if (ctx->needs_input_grad(0)) {
      d_rows = empty({rows.size(0), rows.size(1)}, rows, rows.scalar_type());
    }
    if (ctx->needs_input_grad(1)) {
      d_weights = empty({position.size(0), position.size(1)}, rows, at::kFloat);
    }
    if (rows.numel() > 0) {
      check(bt_combine_backward(
                rows.data_ptr(), grad.data_ptr(), elem_of(rows),
                static_cast<int>(position.size(0)), static_cast<int>(position.size(1)),
                static_cast<int>(rows.size(1)), grad.stride(0), position.data_ptr<int>(),
                offsets.data_ptr<int>() + offsets.numel() - 1, weights.data_ptr<float>(),
                d_rows.defined() ? d_rows.data_ptr() : nullptr,
                d_weights.defined() ? d_weights.data_ptr<float>() : nullptr, place.stream),
            "combine backward");
    } else if (d_weights.defined()) {
      d_weights.zero_();
    }
    return {once(d_rows, saved[1]), once(d_weights, saved[0]), at::Tensor()};
  }
};

// dispatch(x, plan)
PyObject* dispatch(PyObject* const* a) {
  const at::Tensor& x = tensor(a[0], "x");
  rows_of(x, "x");
  const Plan plan = plan_of(a[1], x);
  if (x.size(0) != plan.tokens) {
    refuse("the plan is for ", plan.tokens, " tokens, x has ", x.size(0));
  }
  small(x.size(1), "the width");
  return THPVariable_Wrap(wants_grad(x) ? DispatchNode::apply(x, plan) : dispatch_forward(x, plan));
}

// combine(rows, plan, weights)
PyObject* combine(PyObject* const* a) {
  const at::Tensor& rows = tensor(a[0], "rows");
  rows_of(rows, "rows");
  const Plan plan = plan_of(a[1], rows);
  if (rows.size(0) != static_cast<int64_t>(plan.tokens) * plan.k) {
    refuse("the plan is for ", static_cast<int64_t>(plan.tokens) * plan.k, " rows, got ",
           rows.size(0));
  }
  small(rows.size(1), "the width");
  const at::Tensor& weights = tensor(a[2], "weights");
  if (weights.scalar_type() != at::kFloat || weights.sizes() != plan.position.sizes() ||
      weights.device() != rows.device()) {
    refuse("weights must be a float32 tensor of plan.position's shape on the rows' device");
  }
  const bool for_rows = wants_grad(rows), for_weights = wants_grad(weights);
  if (for_rows || for_weights) {
    return THPVariable_Wrap(CombineNode::apply(rows, weights, plan));
  }
  return THPVariable_Wrap(combine_forward(rows, plan.position, weights.contiguous()));
}

// ---- the module --------------------------------------------------------------------------------

template <PyObject* (*F)(PyObject* const*), Py_ssize_t N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  try {
    if (n != N) {
      PyErr_Format(PyExc_TypeError, "%zd arguments expected, got %zd", N, n);
      return nullptr;
    }
    return F(args);
  } catch (const Refused& r) {
    return raise(r);
  } catch (const Failed& f) {
    return raise(f);
  }
  END_HANDLE_TH_ERRORS
}

template <PyObject* (*F)(PyObject* const*), Py_ssize_t N>
PyMethodDef method(const char* name) {
  return PyMethodDef{name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<F, N>)),
                     METH_FASTCALL, nullptr};
}

PyMethodDef methods[] = {
    method<sample, 7>("sample"),
    method<route, 8>("route"),
    method<expert_order, 2>("expert_order"),
    method<dispatch, 2>("dispatch"),
    method<combine, 3>("combine"),
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensors",
                      "Tensor-level calls of sampling and the experts' operators.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensors() { return PyModule_Create(&module); }
