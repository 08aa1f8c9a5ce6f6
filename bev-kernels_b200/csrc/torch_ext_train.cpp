// torch_ext_train.cpp -- module _bevk_train_ext: the training-side operators
// (group norm with activation on channels-last tensors, embedding lookup with
// scaling, the global gradient norm and clipping) over the C ABI.
#include <c10/cuda/CUDACachingAllocator.h>
#include <torch/csrc/autograd/forward_grad.h>

#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "torch_ext_common.h"

using at::Tensor;
using namespace bevk_ext;

namespace {

using OptTensor = std::optional<Tensor>;

// Counts a write through a tensor's pointer, as torch's own operators count theirs:
// a graph that saved the tensor before then refuses the new values.  (Inference
// tensors are not counted.)
void count_write(const Tensor &t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// The operators have no forward-mode derivative.  A tangent is refused, as torch
// refuses it for a Function without one: the result would have none, which reads
// as a derivative of zero.  (In the forward of a custom Function forward mode is
// off: what is called there has its derivative from the Function.)  Tensors can
// have tangents only within a dual level, which is asked for once a call.
bool tangents_possible() {
  return c10::AutogradState::get_tls_state().get_fw_grad_mode() &&
         torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr;
}
void check_no_tangent(const Tensor &t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(),
                              "bevk: a tensor has a forward-mode tangent; this operator has no "
                              "forward-mode derivative");
}
void check_no_tangents(std::initializer_list<const Tensor *> tensors) {
  if (!tangents_possible()) return;
  for (const Tensor *t : tensors)
    if (t) check_no_tangent(*t);
}
const Tensor *opt_ptr(const OptTensor &t) { return t ? &*t : nullptr; }

// ------------------------------------------------------- group norm + act

// Whether the tensor can be addressed as {image, pixel} strides with channel
// stride 1: the spatial axes flatten, the channels are consecutive.
bool channels_last_rows(const Tensor &t) {
  if (t.size(1) > 1 && t.stride(1) != 1) return false;
  int64_t inner = -1;  // stride that the next outer spatial axis must have
  for (int64_t d = t.dim() - 1; d >= 2; --d) {
    if (t.size(d) == 1) continue;
    if (inner >= 0 && t.stride(d) != inner) return false;
    inner = t.stride(d) * t.size(d);
  }
  return true;
}

// A channels-last tensor of t's shape (any number of spatial axes).
Tensor empty_channels_last(const Tensor &t, at::ScalarType dtype) {
  std::vector<int64_t> sizes = t.sizes().vec(), strides(sizes.size());
  int64_t step = 1;
  strides[1] = 1;
  step = sizes[1];
  for (int64_t d = t.dim() - 1; d >= 2; --d) {
    strides[d] = step;
    step *= sizes[d];
  }
  strides[0] = step;
  return at::empty_strided(sizes, strides, t.options().dtype(dtype));
}

Tensor as_channels_last(const Tensor &t) {
  if (channels_last_rows(t)) return t;
  Tensor out = empty_channels_last(t, t.scalar_type());
  out.copy_(t);
  return out;
}

void row_strides(const Tensor &t, int64_t strides[2]) {
  strides[0] = t.size(0) > 1 ? t.stride(0) : 0;
  strides[1] = 0;
  for (int64_t d = t.dim() - 1; d >= 2; --d)
    if (t.size(d) > 1) {
      strides[1] = t.stride(d);
      break;
    }
  // a single pixel or image is never stepped over
}

const void *ptr(const OptTensor &t) { return t ? t->data_ptr() : nullptr; }

bevk_group_norm_problem gn_problem(const Tensor &input, int64_t num_groups,
                                   const OptTensor &weight, const OptTensor &bias, double eps,
                                   int64_t act) {
  check_cuda(input, "input");
  check_no_tangents({&input, opt_ptr(weight), opt_ptr(bias)});
  TORCH_CHECK(input.dim() >= 2, "bevk: input must be [N, C, *spatial]");
  TORCH_CHECK(num_groups > 0 && input.size(1) > 0 && input.size(1) % num_groups == 0,
              "bevk: num_groups=", str(num_groups), " must divide the channels (",
              str(input.size(1)), ")");
  TORCH_CHECK(input.size(0) < (int64_t(1) << 31) && input.size(1) < (int64_t(1) << 24),
              "bevk: input is too large");
  bevk_group_norm_problem p = {};
  p.dtype = dtype_of(input);
  p.param_dtype = p.dtype;
  bool first = true;
  for (const OptTensor *t : {&weight, &bias}) {
    if (!*t) continue;
    check_same_device(input, **t, "weight / bias");
    TORCH_CHECK((*t)->dim() == 1 && (*t)->size(0) == input.size(1) && (*t)->is_contiguous(),
                "bevk: weight and bias must be contiguous [C]");
    const int dt = dtype_of(**t);
    TORCH_CHECK(first || dt == p.param_dtype, "bevk: weight and bias must share a dtype");
    p.param_dtype = dt;
    first = false;
  }
  p.batch = static_cast<int>(input.size(0));
  p.channels = static_cast<int>(input.size(1));
  p.groups = static_cast<int>(num_groups);
  p.act = static_cast<int>(act);
  p.pixels = 1;
  for (int64_t d = 2; d < input.dim(); ++d) p.pixels *= input.size(d);
  p.eps = static_cast<float>(eps);
  return p;
}

// Scratch memory of the current device and stream, back to torch's allocator at
// the end of the scope (and half the host time of a tensor).
c10::DataPtr scratch(size_t bytes) {
  return c10::cuda::CUDACachingAllocator::get()->allocate(std::max<size_t>(bytes, 1));
}

std::tuple<Tensor, OptTensor, OptTensor> group_norm_act_forward(
    const Tensor &input_, int64_t num_groups, const OptTensor &weight, const OptTensor &bias,
    double eps, int64_t act, bool stats) {
  bevk_group_norm_problem p = gn_problem(input_, num_groups, weight, bias, eps, act);
  const c10::cuda::CUDAGuard guard(input_.device());
  const Tensor input = as_channels_last(input_);
  Tensor output = empty_channels_last(input, input.scalar_type());
  row_strides(input, p.input_strides);
  row_strides(output, p.output_strides);
  OptTensor mean, rstd;
  if (stats) {
    const auto opt = input.options().dtype(at::kFloat);
    mean = at::empty({input.size(0), num_groups}, opt);
    rstd = at::empty({input.size(0), num_groups}, opt);
  }
  const size_t bytes = bevk_group_norm_act_workspace_bytes(&p, 0);
  const c10::DataPtr ws = scratch(bytes);
  check_status(bevk_group_norm_act_forward(
                   &p, input.data_ptr(), ptr(weight), ptr(bias), output.data_ptr(),
                   stats ? mean->data_ptr<float>() : nullptr,
                   stats ? rstd->data_ptr<float>() : nullptr, ws.get(), bytes,
                   current_stream(input)),
               "group_norm_act_forward");
  return {output, mean, rstd};
}

std::tuple<OptTensor, OptTensor, OptTensor> group_norm_act_backward(
    const Tensor &grad_output_, const Tensor &input_, const Tensor &mean, const Tensor &rstd,
    int64_t num_groups, const OptTensor &weight, const OptTensor &bias, int64_t act,
    bool need_input, bool need_weight, bool need_bias) {
  bevk_group_norm_problem p = gn_problem(input_, num_groups, weight, bias, 0.0, act);
  for (const Tensor *t : {&grad_output_, &mean, &rstd})
    check_same_device(input_, *t, "group norm tensor");
  check_no_tangents({&grad_output_, &mean, &rstd});
  TORCH_CHECK(grad_output_.sizes() == input_.sizes() &&
                  grad_output_.scalar_type() == input_.scalar_type(),
              "bevk: grad_output must have input's shape and dtype");
  for (const Tensor *t : {&mean, &rstd})
    TORCH_CHECK(t->scalar_type() == at::kFloat && t->is_contiguous() && t->dim() == 2 &&
                    t->size(0) == input_.size(0) && t->size(1) == num_groups,
                "bevk: mean and rstd must be contiguous fp32 [N, num_groups]");
  const c10::cuda::CUDAGuard guard(input_.device());
  const Tensor input = as_channels_last(input_), grad_output = as_channels_last(grad_output_);
  row_strides(input, p.input_strides);
  row_strides(grad_output, p.grad_output_strides);
  OptTensor gi, gw, gb;
  if (need_input) {
    gi = empty_channels_last(input, input.scalar_type());
    row_strides(*gi, p.output_strides);
  }
  const auto popt = weight ? weight->options() : bias ? bias->options() : input.options();
  if (need_weight) gw = at::empty({input.size(1)}, popt);
  if (need_bias) gb = at::empty({input.size(1)}, popt);
  const size_t bytes = bevk_group_norm_act_workspace_bytes(&p, 1);
  const c10::DataPtr ws = scratch(bytes);
  const auto out = [](const OptTensor &t) { return t ? t->data_ptr() : nullptr; };
  check_status(bevk_group_norm_act_backward(
                   &p, grad_output.data_ptr(), input.data_ptr(), mean.data_ptr<float>(),
                   rstd.data_ptr<float>(), ptr(weight), ptr(bias), out(gi), out(gw), out(gb),
                   ws.get(), bytes, current_stream(input)),
               "group_norm_act_backward");
  return {gi, gw, gb};
}

// ------------------------------------------------------------- embedding

bool wide_ids(const Tensor &ids) {
  TORCH_CHECK(ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt,
              "bevk: ids must be int64 or int32");
  return ids.scalar_type() == at::kLong;
}

// t's rows one after the other, or t where they can be addressed as they are.
Tensor as_rows(const Tensor &t) {
  return t.dim() == 2 && (t.size(1) == 1 || t.stride(1) == 1) && t.stride(0) >= t.size(1)
             ? t
             : t.contiguous();
}
int64_t row_stride(const Tensor &t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

Tensor embedding_forward(const Tensor &table, const Tensor &ids_, double scale) {
  check_cuda(table, "weight");
  check_same_device(table, ids_, "ids");
  check_no_tangents({&table});
  TORCH_CHECK(table.dim() == 2 && table.size(1) > 0, "bevk: weight must be [rows, dim]");
  TORCH_CHECK(table.size(1) < (int64_t(1) << 24), "bevk: weight has too many columns");
  const bool wide = wide_ids(ids_);
  const int dt = dtype_of(table);
  const c10::cuda::CUDAGuard guard(table.device());
  const Tensor rows = as_rows(table), ids = ids_.contiguous();
  std::vector<int64_t> sizes = ids.sizes().vec();
  sizes.push_back(table.size(1));
  Tensor out = at::empty(sizes, table.options());
  check_status(bevk_embedding_forward(rows.data_ptr(), row_stride(rows), ids.data_ptr(), wide,
                                      ids.numel(), rows.size(0), static_cast<int>(rows.size(1)),
                                      static_cast<float>(scale), out.data_ptr(), dt,
                                      current_stream(table)),
               "embedding_forward");
  return out;
}

// Where `into` is given the gradient is added to it (and it is returned).
Tensor embedding_backward(const Tensor &grad_output, const Tensor &ids_, int64_t num_rows,
                          double scale, int64_t padding_idx, const OptTensor &into) {
  check_cuda(grad_output, "grad_output");
  check_same_device(grad_output, ids_, "ids");
  check_no_tangents({&grad_output, opt_ptr(into)});
  const bool wide = wide_ids(ids_);
  TORCH_CHECK(grad_output.dim() == ids_.dim() + 1 &&
                  grad_output.sizes().slice(0, ids_.dim()) == ids_.sizes(),
              "bevk: grad_output must be [*ids.shape, dim]");
  const int64_t dim = grad_output.size(-1);
  TORCH_CHECK(dim > 0 && dim < (int64_t(1) << 24) && num_rows >= 0,
              "bevk: bad number of rows or columns");
  bevk_embedding_backward_args a = {};
  a.grad_output_dtype = dtype_of(grad_output);
  const c10::cuda::CUDAGuard guard(grad_output.device());
  const Tensor ids = ids_.contiguous();
  const Tensor dy = as_rows(grad_output.dim() == 2 ? grad_output : grad_output.reshape({-1, dim}));
  Tensor out;
  if (into) {
    check_same_device(grad_output, *into, "grad_weight");
    TORCH_CHECK(into->dim() == 2 && into->size(0) == num_rows && into->size(1) == dim,
                "bevk: grad_weight must be [num_embeddings, dim]");
    TORCH_CHECK((dim == 1 || into->stride(1) == 1) &&
                    (num_rows <= 1 || into->stride(0) >= dim),
                "bevk: grad_weight's rows must be contiguous and apart");
    out = *into;
  } else {
    out = at::empty({num_rows, dim}, grad_output.options());
  }
  a.grad_table_dtype = dtype_of(out);
  a.num_ids = ids.numel();
  a.num_rows = num_rows;
  a.dim = static_cast<int>(dim);
  a.ids_are_64bit = wide;
  a.grad_output_ld = dy.size(0) > 0 ? row_stride(dy) : dim;
  a.grad_table_ld = num_rows > 0 ? row_stride(out) : dim;
  a.padding_idx = padding_idx;
  a.scale = static_cast<float>(scale);
  a.accumulate = into.has_value();
  const size_t bytes = bevk_embedding_backward_workspace_bytes(&a);
  const c10::DataPtr ws = scratch(bytes);
  check_status(bevk_embedding_backward(&a, dy.data_ptr(), ids.data_ptr(), out.data_ptr(),
                                       ws.get(), bytes, current_stream(grad_output)),
               "embedding_backward");
  if (into) count_write(out);
  return out;
}

// ------------------------------------------------ gradient norm and clipping

bool dense(const Tensor &t) { return t.is_non_overlapping_and_dense(); }

// A dense tensor of like's strides (contiguous where like has holes).
Tensor empty_dense(const Tensor &like, at::ScalarType dtype) {
  return dense(like) ? at::empty_strided(like.sizes(), like.strides(), like.options().dtype(dtype))
                     : at::empty(like.sizes(), like.options().dtype(dtype));
}

// The norm of all tensors; where max_norm is given, also scales them, into
// `out` or in place.  Tensors with holes, and outputs of another layout than
// their gradient's, go through a dense copy.
Tensor grad_clip(const std::vector<Tensor> &grads, std::optional<double> max_norm, double eps,
                 bool inf_norm, const std::optional<std::vector<Tensor>> &out) {
  const at::NoGradGuard no_grad;  // the copies below are no part of the caller's graph
  TORCH_CHECK(!grads.empty(), "bevk: no gradients");
  TORCH_CHECK(!out || out->size() == grads.size(), "bevk: one output for each gradient");
  if (tangents_possible()) {
    for (const Tensor &t : grads) check_no_tangent(t);
    if (max_norm && out)
      for (const Tensor &t : *out) check_no_tangent(t);
  }
  const Tensor &first = grads[0];
  std::vector<bevk_grad_tensor> items(grads.size());
  std::vector<Tensor> keep;                          // copies the call reads or writes
  std::vector<std::pair<Tensor, Tensor>> copy_back;  // (to, from)
  const c10::cuda::OptionalCUDAGuard guard(first.is_cuda() ? std::optional<c10::Device>(first.device())
                                                           : std::nullopt);
  for (size_t i = 0; i < grads.size(); ++i) {
    const Tensor &g = grads[i];
    if (g.device() != first.device() || !g.is_cuda()) {
      check_cuda(g, "gradient");
      check_same_device(first, g, "gradient");
    }
    TORCH_CHECK(g.layout() == at::kStrided, "bevk: gradients must be strided tensors");
    bevk_grad_tensor &it = items[i];
    it.grad_dtype = dtype_of(g);
    it.numel = g.numel();
    if (g.is_contiguous() && (!max_norm || !out)) {  // the common cases, without copies
      it.grad = it.out = g.data_ptr();
      it.out_dtype = it.grad_dtype;
      continue;
    }
    if (g.is_contiguous() && (*out)[i].is_contiguous() && (*out)[i].sizes() == g.sizes() &&
        (*out)[i].device() == g.device()) {
      it.grad = g.data_ptr();
      it.out = (*out)[i].data_ptr();
      it.out_dtype = dtype_of((*out)[i]);
      continue;
    }
    Tensor src = g;
    if (!max_norm) {
      if (!dense(src)) keep.push_back(src = src.contiguous());
      it.grad = it.out = src.data_ptr();
      it.out_dtype = it.grad_dtype;
      continue;
    }
    const Tensor &o = out ? (*out)[i] : g;
    if (out) {
      check_same_device(first, o, "output");
      TORCH_CHECK(o.sizes() == g.sizes(), "bevk: an output must have its gradient's shape");
    }
    for (int64_t d = 0; d < o.dim(); ++d)
      TORCH_CHECK(o.numel() == 0 || o.size(d) == 1 || o.stride(d) != 0,
                  "bevk: an expanded tensor cannot be written");
    const bool in_place = o.data_ptr() == g.data_ptr() && o.scalar_type() == g.scalar_type() &&
                          o.strides() == g.strides();
    Tensor dst = o;
    if (!dense(dst)) {
      keep.push_back(dst = empty_dense(o, o.scalar_type()));
      copy_back.emplace_back(o, dst);
    }
    if (in_place) {
      if (!dst.is_same(o)) {
        dst.copy_(src);
        src = dst;
      }
    } else if (!dense(src) || src.strides() != dst.strides()) {
      Tensor c = empty_dense(dst, src.scalar_type());
      c.copy_(src);
      keep.push_back(src = c);
    }
    it.grad = src.data_ptr();
    it.out = dst.data_ptr();
    it.out_dtype = dtype_of(dst);
  }
  Tensor norm = at::empty({}, first.options().dtype(at::kFloat));
  const size_t bytes = bevk_grad_clip_workspace_bytes(static_cast<int>(items.size()));
  const c10::DataPtr ws = scratch(bytes);
  check_status(bevk_grad_clip(items.data(), static_cast<int>(items.size()),
                              inf_norm ? BEVK_NORM_INF : BEVK_NORM_L2,
                              static_cast<float>(max_norm.value_or(0.0)), static_cast<float>(eps),
                              max_norm.has_value(), norm.data_ptr<float>(), ws.get(), bytes,
                              current_stream(first)),
               "grad_clip");
  for (auto &c : copy_back) c.first.copy_(c.second);
  if (max_norm)
    for (const Tensor &t : out ? *out : grads) count_write(t);
  return norm;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("group_norm_act_forward", &group_norm_act_forward);
  m.def("group_norm_act_backward", &group_norm_act_backward);
  m.def("embedding_forward", &embedding_forward);
  m.def("embedding_backward", &embedding_backward);
  m.def("grad_clip", &grad_clip);
}
