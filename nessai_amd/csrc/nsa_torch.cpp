// torch operators over the C entry points of nsa_grad_norm.hip, nsa_group_norm.hip and nsa_embedding.hip
// (torch.ops.nessai_amd.*; nessai_amd/ops_context.py documents them).  In C++ because their calls are short: a minibatch's
// group norm runs for 5 us on the device and took 130 us, forward and backward, with the checks, allocations and the
// autograd node in Python; clipping 300 gradients spent 220 us reading their attributes.
//
// Nothing here computes.  The public operators check their arguments and record for autograd; each calls one of the inner
// ones (a leading underscore), which exist for the CUDA (ROCm) dispatch key - results and workspaces are allocated and one
// entry point called on the current stream of the tensors' device - and for the Meta key, where they return the results'
// shapes.  The public ones have one body for every key, so a tracer (torch.compile, make_fx) sees the inner ones; those check
// by themselves what the kernels rely on, because a traced graph calls them with tensors of its own.
// The entry points' addresses come from the loaded libnessai_amd.so (nessai_amd/lib.py).
#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <optional>
#include <tuple>
#include <utility>
#include <vector>

#include "../../include/nessai_amd.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct EntryPoints {
  decltype(&nsa_last_error) last_error = nullptr;
  decltype(&nsa_grad_norm_workspace) grad_norm_workspace;
  decltype(&nsa_grad_norm) grad_norm;
  decltype(&nsa_grad_clip) grad_clip;
  decltype(&nsa_group_norm_workspace) group_norm_workspace;
  decltype(&nsa_group_norm_forward) group_norm_forward;
  decltype(&nsa_group_norm_backward) group_norm_backward;
  decltype(&nsa_embedding_forward) embedding_forward;
  decltype(&nsa_embedding_workspace) embedding_workspace;
  decltype(&nsa_embedding_backward) embedding_backward;
};
EntryPoints g_entry;

void bind_library(at::IntArrayRef a) {  // in the order of the struct
  TORCH_CHECK(a.size() == sizeof(EntryPoints) / sizeof(void*), "nessai_amd: wrong number of entry points");
  for (size_t i = 0; i < a.size(); ++i) reinterpret_cast<void**>(&g_entry)[i] = reinterpret_cast<void*>(a[i]);
}

void check(int rc, const char* what) {
  TORCH_CHECK(rc == NSA_OK, what, " failed (code ", rc, "): ", g_entry.last_error());
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

int dtype_code(const Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case at::kFloat: return NSA_DT_F32;
    case at::kBFloat16: return NSA_DT_BF16;
    case at::kHalf: return NSA_DT_F16;
    default:
      TORCH_CHECK_TYPE(false, what, " must be float32, bfloat16 or float16 (got ", t.scalar_type(),
                       "): there is no kernel for other types, and nothing is cast down silently");
  }
}

void on_device(const Tensor& t, const char* what) {
  TORCH_CHECK(t.is_cuda() || t.is_meta(), what, ": nessai_amd operators take tensors on a ROCm device (got ", t.device(),
              "); there is no CPU fallback");
}

Tensor workspace(const Tensor& like, size_t bytes) {
  return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
}

// An inner operator, looked up once by its caller.  Called below autograd's keys: its fallback for operators without a
// derivative puts the arguments on a stack, 25 ns for each tensor of a list.
template <typename F>
struct Inner {
  c10::TypedOperatorHandle<F> handle;
  explicit Inner(const char* name) : handle(c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>()) {}
  template <typename... A>
  auto operator()(A&&... a) const {
    const at::AutoDispatchBelowADInplaceOrView below;
    return handle.call(std::forward<A>(a)...);
  }
};

std::optional<Tensor> given(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

// what a kernel relies on, in an inner operator
void expect(bool holds, const char* what, const char* condition) {
  TORCH_CHECK(holds, "nessai_amd::", what, ": expected ", condition);
}

const void* data(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* mutable_data(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }

bool wants_grad(std::initializer_list<const Tensor*> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : tensors)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// A tangent (forward-mode differentiation) would be lost: results are allocated here, outside torch's own derivatives.
void no_tangent(const Tensor& t, const char* what) {
  TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), what,
              " has no forward-mode derivative: it was given a tensor with a tangent (torch.autograd.forward_ad, torch.func.jvp)");
}

void once(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, " is differentiable once: its backward pass records no graph (create_graph)");
}

// -- group norm with an activation ------------------------------------------------------------------------------------

struct Rows {  // of a contiguous channels-last tensor
  int64_t samples, length, channels;
  explicit Rows(const Tensor& x) : samples(x.size(0)), length(1), channels(x.size(-1)) {
    for (int64_t d = 1; d + 1 < x.dim(); ++d) length *= x.size(d);
  }
};

int param_dtype(const Tensor& weight, const Tensor& bias) {
  const Tensor& p = weight.defined() ? weight : bias;
  return p.defined() ? dtype_code(p, "group_norm_act: weight") : NSA_DT_F32;
}

void expect_group_norm(const Tensor& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias,
                       int64_t groups, const char* what) {
  expect(x.dim() >= 2 && x.is_contiguous(), what, "a contiguous x of two dimensions or more");
  const int64_t channels = x.size(-1);
  expect(groups >= 1 && channels >= 1 && channels <= (1 << 30) && channels % groups == 0, what, "channels in whole groups");
  for (const auto* p : {&weight, &bias})
    if (p->has_value())
      expect((*p)->is_contiguous() && (*p)->dim() == 1 && (*p)->size(0) == channels && (*p)->device() == x.device() &&
                 ((*p)->scalar_type() == at::kFloat || (*p)->scalar_type() == x.scalar_type()),
             what, "a contiguous weight and bias of x's channels, on its device, in float32 or its type");
  expect(!weight.has_value() || !bias.has_value() || weight->scalar_type() == bias->scalar_type(), what,
         "a weight and a bias of one type");
}

std::tuple<Tensor, Tensor> group_norm_results(const Tensor& x, int64_t groups) {
  return {at::empty(x.sizes(), x.options()), at::empty({2, Rows(x).samples, groups}, x.options().dtype(at::kFloat))};
}

// y, and the statistics: [mean, 1 / sqrt(var + eps)][sample][group]
std::tuple<Tensor, Tensor> group_norm_forward(const Tensor& x, const std::optional<Tensor>& weight_,
                                              const std::optional<Tensor>& bias_, int64_t groups, double eps,
                                              int64_t activation) {
  expect_group_norm(x, weight_, bias_, groups, "_group_norm_forward");
  const Rows r(x);
  const Tensor weight = weight_.value_or(Tensor()), bias = bias_.value_or(Tensor());
  auto results = group_norm_results(x, groups);
  const auto& [y, stats] = results;
  if (x.numel() == 0) return results;
  const c10::DeviceGuard guard(x.device());
  const int code = dtype_code(x, "group_norm_act: x");
  const size_t size = g_entry.group_norm_workspace(r.samples, r.length, r.channels, groups, code, 0);
  const Tensor ws = workspace(x, size);
  float* mean = (float*)stats.mutable_data_ptr();
  check(g_entry.group_norm_forward(r.samples, r.length, r.channels, groups, code, data(x), param_dtype(weight, bias),
                                   data(weight), data(bias), (float)eps, activation, y.mutable_data_ptr(), mean,
                                   mean + r.samples * groups, ws.mutable_data_ptr(), size, stream_of(x)),
        "nsa_group_norm_forward");
  return results;
}

std::tuple<Tensor, Tensor> group_norm_forward_meta(const Tensor& x, const std::optional<Tensor>& weight,
                                                   const std::optional<Tensor>& bias, int64_t groups, double, int64_t) {
  expect_group_norm(x, weight, bias, groups, "_group_norm_forward");
  return group_norm_results(x, groups);
}

// dx, dweight, dbias: undefined where they are not wanted
std::tuple<Tensor, Tensor, Tensor> group_norm_gradients(const Tensor& dy, const Tensor& x, const std::optional<Tensor>& weight,
                                                        const std::optional<Tensor>& bias, const Tensor& stats, int64_t groups,
                                                        int64_t, std::array<bool, 3> wanted) {
  const char* what = "_group_norm_backward";
  expect_group_norm(x, weight, bias, groups, what);
  expect(dy.is_contiguous() && dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type() && dy.device() == x.device(),
         what, "a contiguous dy of x's shape, type and device");
  expect(stats.is_contiguous() && stats.numel() == 2 * x.size(0) * groups && stats.scalar_type() == at::kFloat &&
             stats.device() == x.device(),
         what, "the forward pass's statistics");
  auto like = [](bool want, const std::optional<Tensor>& t) {
    return want && t.has_value() ? at::empty(t->sizes(), t->options()) : Tensor();
  };
  return {like(wanted[0], x), like(wanted[1], weight), like(wanted[2], bias)};
}

std::tuple<Tensor, Tensor, Tensor> group_norm_backward(const Tensor& dy, const Tensor& x, const std::optional<Tensor>& weight_,
                                                       const std::optional<Tensor>& bias_, const Tensor& stats,
                                                       int64_t groups, int64_t activation, std::array<bool, 3> wanted) {
  auto results = group_norm_gradients(dy, x, weight_, bias_, stats, groups, activation, wanted);
  const Rows r(x);
  const Tensor weight = weight_.value_or(Tensor()), bias = bias_.value_or(Tensor());
  const c10::DeviceGuard guard(x.device());
  const auto& [dx, dw, db] = results;
  const int code = dtype_code(x, "group_norm_act: x");
  const size_t size = g_entry.group_norm_workspace(r.samples, r.length, r.channels, groups, code, 1);
  const Tensor ws = workspace(x, size);
  const float* mean = (const float*)stats.const_data_ptr();
  check(g_entry.group_norm_backward(r.samples, r.length, r.channels, groups, code, data(x), data(dy),
                                    param_dtype(weight, bias), data(weight), data(bias), activation, mean,
                                    mean + r.samples * groups, mutable_data(dx), mutable_data(dw), mutable_data(db),
                                    ws.mutable_data_ptr(), size, stream_of(x)),
        "nsa_group_norm_backward");
  return results;
}

std::tuple<Tensor, Tensor> call_group_norm_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, int64_t groups,
                                                   double eps, int64_t activation) {
  static const Inner<decltype(group_norm_forward)> op("nessai_amd::_group_norm_forward");
  return op(x, given(weight), given(bias), groups, eps, activation);
}

struct GroupNormAct : public torch::autograd::Function<GroupNormAct> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& weight_,
                        const std::optional<Tensor>& bias_, int64_t groups, double eps, int64_t activation) {
    const Tensor weight = weight_.value_or(Tensor()), bias = bias_.value_or(Tensor());
    auto [y, stats] = call_group_norm_forward(x, weight, bias, groups, eps, activation);
    ctx->save_for_backward({x, weight, bias, stats});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["activation"] = activation;
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("group_norm_act");
    static const Inner<decltype(group_norm_backward)> op("nessai_amd::_group_norm_backward");
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &bias = saved[2], &stats = saved[3];
    std::array<bool, 3> wanted = {};
    size_t edge = 0;  // of the tensors that were given, in order
    wanted[0] = ctx->needs_input_grad(edge++);
    wanted[1] = weight.defined() && ctx->needs_input_grad(edge++);
    wanted[2] = bias.defined() && ctx->needs_input_grad(edge++);
    auto [dx, dw, db] = op(grads[0].contiguous(), x, given(weight), given(bias), stats, ctx->saved_data["groups"].toInt(),
                           ctx->saved_data["activation"].toInt(), wanted);
    return {dx, dw, db, Tensor(), Tensor(), Tensor()};
  }
};

Tensor group_norm_act(const Tensor& x_, int64_t groups, const std::optional<Tensor>& weight_,
                      const std::optional<Tensor>& bias_, double eps, int64_t activation) {
  TORCH_CHECK_VALUE(x_.dim() >= 2, "expected a tensor of shape (N, ..., C), got ", x_.sizes());
  dtype_code(x_, "group_norm_act: x");
  const int64_t channels = x_.size(-1);
  TORCH_CHECK_VALUE(groups >= 1 && channels >= 1 && channels % groups == 0, channels,
                    " channels cannot be divided into ", groups, " groups");
  TORCH_CHECK_VALUE(channels <= (1 << 30), "group_norm_act: at most 2**30 channels (got ", channels, ")");
  TORCH_CHECK_VALUE(eps >= 0.0, "eps must not be negative (got ", eps, ")");
  Tensor weight = weight_.value_or(Tensor()), bias = bias_.value_or(Tensor());
  for (const Tensor* t : {&x_, &std::as_const(weight), &std::as_const(bias)}) no_tangent(*t, "group_norm_act");
  const char* names[] = {"weight", "bias"};
  Tensor* params[] = {&weight, &bias};
  for (int i = 0; i < 2; ++i) {
    Tensor& p = *params[i];
    if (!p.defined()) continue;
    TORCH_CHECK_VALUE(p.dim() == 1 && p.size(0) == channels, "expected a ", names[i], " of shape (", channels, ",), got ", p.sizes());
    TORCH_CHECK_TYPE(p.scalar_type() == at::kFloat || p.scalar_type() == x_.scalar_type(), "group_norm_act: ", names[i],
                     " must be float32 or of x's type ", x_.scalar_type(), " (got ", p.scalar_type(), ")");
    TORCH_CHECK_VALUE(p.device() == x_.device(), "group_norm_act: ", names[i], " is on ", p.device(), ", x on ", x_.device());
    p = p.contiguous();
  }
  TORCH_CHECK_TYPE(!weight.defined() || !bias.defined() || weight.scalar_type() == bias.scalar_type(),
                   "group_norm_act: weight and bias must have one type");
  on_device(x_, "group_norm_act");
  const Tensor x = x_.contiguous();
  if (wants_grad({&x, &weight, &bias})) return GroupNormAct::apply(x, given(weight), given(bias), groups, eps, activation);
  return std::get<0>(call_group_norm_forward(x, weight, bias, groups, eps, activation));
}

// -- embedding --------------------------------------------------------------------------------------------------------

Tensor embedding_rows(const Tensor& ids, const Tensor& weight, double) {
  expect(ids.is_contiguous() && (ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong), "_embedding_forward",
         "contiguous int32 or int64 indices");
  expect(weight.is_contiguous() && weight.dim() == 2 && weight.device() == ids.device(), "_embedding_forward",
         "a contiguous table on the indices' device");
  std::vector<int64_t> shape = ids.sizes().vec();
  shape.push_back(weight.size(1));
  return at::empty(shape, weight.options());
}

Tensor embedding_forward(const Tensor& ids, const Tensor& weight, double scale) {
  Tensor out = embedding_rows(ids, weight, scale);
  if (out.numel() == 0) return out;
  const c10::DeviceGuard guard(weight.device());
  check(g_entry.embedding_forward(ids.numel(), weight.size(0), weight.size(1), dtype_code(weight, "embedding: weight"),
                                  data(ids), (int)ids.element_size(), data(weight), (float)scale, out.mutable_data_ptr(),
                                  stream_of(weight)),
        "nsa_embedding_forward");
  return out;
}

Tensor embedding_table(const Tensor& dy, const Tensor& ids, int64_t vocab, int64_t width, double, int64_t) {
  expect(ids.is_contiguous() && (ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong), "_embedding_backward",
         "contiguous int32 or int64 indices");
  expect(vocab >= 1 && width >= 1 && width <= (1 << 20) && dy.is_contiguous() && dy.numel() == ids.numel() * width &&
             dy.device() == ids.device(),
         "_embedding_backward", "a contiguous dy of a row for each index, on their device");
  return at::empty({vocab, width}, dy.options());
}

Tensor embedding_backward(const Tensor& dy, const Tensor& ids, int64_t vocab, int64_t width, double scale, int64_t padding) {
  const c10::DeviceGuard guard(dy.device());
  Tensor dweight = embedding_table(dy, ids, vocab, width, scale, padding);
  const int code = dtype_code(dy, "embedding: weight");
  const size_t size = g_entry.embedding_workspace(ids.numel(), vocab, width, code);
  const Tensor ws = workspace(dy, size);
  check(g_entry.embedding_backward(ids.numel(), vocab, width, code, data(ids), (int)ids.element_size(), data(dy), (float)scale,
                                   padding, dweight.mutable_data_ptr(), ws.mutable_data_ptr(), size, stream_of(dy)),
        "nsa_embedding_backward");
  return dweight;
}

Tensor call_embedding_forward(const Tensor& ids, const Tensor& weight, double scale) {
  static const Inner<decltype(embedding_forward)> op("nessai_amd::_embedding_forward");
  return op(ids, weight, scale);
}

struct Embedding : public torch::autograd::Function<Embedding> {
  static Tensor forward(AutogradContext* ctx, const Tensor& weight, const Tensor& ids, double scale, int64_t padding) {
    ctx->save_for_backward({ids});
    ctx->saved_data["vocab"] = weight.size(0);
    ctx->saved_data["width"] = weight.size(1);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    return call_embedding_forward(ids, weight, scale);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("embedding");
    static const Inner<decltype(embedding_backward)> op("nessai_amd::_embedding_backward");
    const Tensor ids = ctx->get_saved_variables()[0];
    return {op(grads[0].contiguous(), ids, ctx->saved_data["vocab"].toInt(), ctx->saved_data["width"].toInt(),
               ctx->saved_data["scale"].toDouble(), ctx->saved_data["padding"].toInt()),
            Tensor(), Tensor(), Tensor()};
  }
};

Tensor embedding(const Tensor& ids_, const Tensor& weight_, double scale, std::optional<int64_t> padding_idx) {
  TORCH_CHECK_TYPE(ids_.scalar_type() == at::kInt || ids_.scalar_type() == at::kLong,
                   "embedding: indices must be int32 or int64 (got ", ids_.scalar_type(), ")");
  TORCH_CHECK_VALUE(weight_.dim() == 2 && weight_.size(0) >= 1 && weight_.size(1) >= 1,
                    "embedding: expected a table of shape (V, D), got ", weight_.sizes());
  dtype_code(weight_, "embedding: weight");
  no_tangent(weight_, "embedding");
  const int64_t vocab = weight_.size(0), most = (1LL << 31) - 1;
  TORCH_CHECK_VALUE(vocab <= most && ids_.numel() <= most && weight_.size(1) <= (1 << 20),
                    "embedding: at most 2**31 - 1 rows and indices and 2**20 columns");
  int64_t padding = -1;
  if (padding_idx.has_value()) {
    TORCH_CHECK_VALUE(-vocab <= *padding_idx && *padding_idx < vocab, "embedding: padding_idx ", *padding_idx,
                      " is outside a table of ", vocab, " rows");
    padding = *padding_idx < 0 ? *padding_idx + vocab : *padding_idx;
  }
  TORCH_CHECK_VALUE(ids_.device() == weight_.device(), "embedding: indices are on ", ids_.device(), ", weight on ", weight_.device());
  on_device(weight_, "embedding");
  const Tensor ids = ids_.contiguous(), weight = weight_.contiguous();
  return wants_grad({&weight}) ? Embedding::apply(weight, ids, scale, padding) : call_embedding_forward(ids, weight, scale);
}

// -- the norm over many gradients, and the clip -----------------------------------------------------------------------

void check_gradients(const std::vector<Tensor>& tensors, const char* what) {
  for (const Tensor& t : tensors) {
    TORCH_CHECK_TYPE(t.layout() == at::kStrided, what, ": gradients must be dense (got ", t.layout(), ")");
    dtype_code(t, what);
    no_tangent(t, what);
    TORCH_CHECK_VALUE(t.device() == tensors[0].device(), what, ": gradients on several devices: ", tensors[0].device(), ", ", t.device());
  }
  on_device(tensors[0], what);
}

void expect_dense(at::TensorList tensors, const char* what) {
  for (const Tensor& t : tensors)
    expect(t.is_non_overlapping_and_dense() && t.device() == tensors[0].device(), what, "dense tensors on one device");
}

// clip: by max_norm, in place; otherwise the norm alone.  Every tensor fills one stretch of memory.
Tensor norm_call(at::TensorList tensors, int64_t kind, bool clip, double max_norm) {
  expect_dense(tensors, clip ? "_clip_gradients_" : "_total_norm");
  const c10::DeviceGuard guard(tensors[0].device());
  const int count = (int)tensors.size();
  std::vector<void*> places(count);
  std::vector<long long> sizes(count);
  std::vector<int> codes(count);
  long long elements = 0;
  for (int i = 0; i < count; ++i) {
    const Tensor& t = tensors[i];
    // (what is written is asked for as such: a lazy clone then gets memory of its own; the norm only reads)
    places[i] = clip ? t.mutable_data_ptr() : const_cast<void*>(t.const_data_ptr());
    sizes[i] = t.numel();
    elements += sizes[i];
    codes[i] = dtype_code(t, "gradients");
  }
  Tensor out = at::empty({}, tensors[0].options().dtype(at::kFloat));
  const size_t size = g_entry.grad_norm_workspace(count, elements);
  const Tensor ws = workspace(out, size);
  if (clip)
    check(g_entry.grad_clip(count, places.data(), sizes.data(), codes.data(), kind, (float)max_norm, ws.mutable_data_ptr(),
                            size, (float*)out.mutable_data_ptr(), stream_of(out)),
          "nsa_grad_clip");
  else
    check(g_entry.grad_norm(count, places.data(), sizes.data(), codes.data(), kind, ws.mutable_data_ptr(), size,
                            (float*)out.mutable_data_ptr(), stream_of(out)),
          "nsa_grad_norm");
  return out;
}

Tensor total_norm(at::TensorList tensors, int64_t kind) { return norm_call(tensors, kind, false, 0.0); }
Tensor clip_gradients(at::TensorList tensors, int64_t kind, double max_norm) { return norm_call(tensors, kind, true, max_norm); }
Tensor total_norm_meta(at::TensorList tensors, int64_t) {
  expect_dense(tensors, "_total_norm");
  return at::empty({}, tensors[0].options().dtype(at::kFloat));
}
Tensor clip_gradients_meta(at::TensorList tensors, int64_t kind, double) { return total_norm_meta(tensors, kind); }

Tensor call_total_norm(at::TensorList tensors, int64_t kind) {
  static const Inner<decltype(total_norm)> op("nessai_amd::_total_norm");
  return op(tensors, kind);
}

Tensor grad_norm(at::TensorList tensors, int64_t kind) {
  if (tensors.empty()) return at::zeros({}, at::kFloat);
  const at::NoGradGuard no_grad;
  std::vector<Tensor> grads = tensors.vec();
  check_gradients(grads, "grad_norm: gradients");
  for (Tensor& g : grads)
    if (!g.is_non_overlapping_and_dense()) g = g.contiguous();
  return call_total_norm(grads, kind);
}

Tensor clip_(std::vector<Tensor> grads, int64_t kind, double max_norm, bool error_if_nonfinite) {
  TORCH_CHECK_VALUE(max_norm >= 0.0, "max_norm must not be negative or NaN (got ", max_norm, ")");
  if (grads.empty()) return at::zeros({}, at::kFloat);
  const at::NoGradGuard no_grad;
  check_gradients(grads, "clip_grad_norm_: gradients");
  // a gradient with gaps between its elements is clipped in a copy; one whose elements share memory cannot be
  std::vector<Tensor> dense = grads;
  bool copies = false;
  for (Tensor& g : dense) {
    if (g.is_non_overlapping_and_dense()) continue;
    copies = true;
    for (int64_t d = 0; d < g.dim(); ++d)
      TORCH_CHECK_VALUE(g.stride(d) != 0 || g.size(d) <= 1,
                        "clip_grad_norm_: a gradient's elements overlap in memory (an expanded tensor); clone it");
    g = g.contiguous();
  }
  if (copies) {  // (the entry point sees those, not what they are copies of: one gradient given twice would pass)
    std::vector<std::pair<const void*, int64_t>> first;
    for (const Tensor& g : grads)
      if (g.numel() > 0) first.emplace_back(g.storage().unsafeGetStorageImpl(), g.storage_offset());
    std::sort(first.begin(), first.end());
    TORCH_CHECK(std::adjacent_find(first.begin(), first.end()) == first.end(), "clip_grad_norm_: two gradients overlap in memory");
  }
  if (error_if_nonfinite)
    TORCH_CHECK(std::isfinite(call_total_norm(dense, kind).item<float>()),
                "The total norm of the gradients from `parameters` is non-finite, so it cannot be clipped");
  static const Inner<decltype(clip_gradients)> op("nessai_amd::_clip_gradients_");
  const Tensor norm = op(dense, kind, max_norm);
  for (size_t i = 0; i < grads.size(); ++i) {
    if (!dense[i].is_same(grads[i])) grads[i].copy_(dense[i]);
    // the kernels wrote behind torch's back: graphs that saved a gradient must see that it changed
    else if (!grads[i].is_inference()) grads[i].unsafeGetTensorImpl()->bump_version();
  }
  return norm;
}

Tensor clip_grad_norm(at::TensorList parameters, int64_t kind, double max_norm, bool error_if_nonfinite) {
  std::vector<Tensor> grads;
  grads.reserve(parameters.size());
  for (const Tensor& p : parameters)
    if (p.grad().defined()) grads.push_back(p.grad());
  return clip_(std::move(grads), kind, max_norm, error_if_nonfinite);
}

// the same of the gradients themselves: a tracer, whose stand-ins for the parameters have no gradients, sees what changes
Tensor clip_grad_norm_of(at::TensorList gradients, int64_t kind, double max_norm, bool error_if_nonfinite) {
  return clip_(gradients.vec(), kind, max_norm, error_if_nonfinite);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(nessai_amd, m) {
  m.def("_bind_library(int[] addresses) -> ()", &bind_library);
  m.def("group_norm_act(Tensor x, int num_groups, Tensor? weight, Tensor? bias, float eps, int activation) -> Tensor",
        &group_norm_act);
  m.def("_group_norm_forward(Tensor x, Tensor? weight, Tensor? bias, int num_groups, float eps, int activation) -> "
        "(Tensor, Tensor)");
  m.def("_group_norm_backward(Tensor dy, Tensor x, Tensor? weight, Tensor? bias, Tensor stats, int num_groups, "
        "int activation, bool[3] wanted) -> (Tensor, Tensor, Tensor)");
  m.def("embedding(Tensor indices, Tensor weight, float scale, int? padding_idx) -> Tensor", &embedding);
  m.def("_embedding_forward(Tensor indices, Tensor weight, float scale) -> Tensor");
  m.def("_embedding_backward(Tensor dy, Tensor indices, int rows, int width, float scale, int padding) -> Tensor");
  m.def("grad_norm(Tensor[] tensors, int kind) -> Tensor", &grad_norm);
  m.def("_total_norm(Tensor[] tensors, int kind) -> Tensor");
  m.def("clip_grad_norm_(Tensor[] parameters, int kind, float max_norm, bool error_if_nonfinite) -> Tensor",
        &clip_grad_norm);
  m.def("clip_grad_norm_of_(Tensor(a!)[] gradients, int kind, float max_norm, bool error_if_nonfinite) -> Tensor",
        &clip_grad_norm_of);
  m.def("_clip_gradients_(Tensor(a!)[] gradients, int kind, float max_norm) -> Tensor");
}

TORCH_LIBRARY_IMPL(nessai_amd, CUDA, m) {
  m.impl("_group_norm_forward", &group_norm_forward);
  m.impl("_group_norm_backward", &group_norm_backward);
  m.impl("_embedding_forward", &embedding_forward);
  m.impl("_embedding_backward", &embedding_backward);
  m.impl("_total_norm", &total_norm);
  m.impl("_clip_gradients_", &clip_gradients);
}

TORCH_LIBRARY_IMPL(nessai_amd, Meta, m) {
  m.impl("_group_norm_forward", &group_norm_forward_meta);
  m.impl("_group_norm_backward", &group_norm_gradients);
  m.impl("_embedding_forward", &embedding_rows);
  m.impl("_embedding_backward", &embedding_table);
  m.impl("_total_norm", &total_norm_meta);
  m.impl("_clip_gradients_", &clip_gradients_meta);
}
