// bevk_train_api.cu -- the extern "C" entry points of the training-side
// operators declared in include/bevk.h: argument validation and dispatch.  No
// entry point allocates device memory.
#include <cuda_runtime.h>

#include <cmath>

#include "bevk.h"
#include "bevk_internal.h"

using namespace bevk;

namespace {

bool known_dtype(int dtype) {
  return dtype == BEVK_DTYPE_F32 || dtype == BEVK_DTYPE_F16 || dtype == BEVK_DTYPE_BF16;
}

// Checks a group norm problem; `backward` also looks at grad_output's strides.
int check_group_norm(const bevk_group_norm_problem *p, bool backward) {
  if (!p) return fail(BEVK_ERR_INVALID_ARGUMENT, "group_norm_act: null problem");
  if (!known_dtype(p->dtype))
    return fail(BEVK_ERR_UNSUPPORTED, "group_norm_act: dtype %d (f32, f16, bf16)", p->dtype);
  if (p->param_dtype != p->dtype && p->param_dtype != BEVK_DTYPE_F32)
    return fail(BEVK_ERR_UNSUPPORTED,
                "group_norm_act: parameter dtype must be the tensors' dtype or f32");
  if (p->batch < 0 || p->pixels < 0 || p->channels <= 0 || p->groups <= 0)
    return fail(BEVK_ERR_INVALID_ARGUMENT, "group_norm_act: bad sizes");
  if (p->channels % p->groups)
    return fail(BEVK_ERR_INVALID_ARGUMENT, "group_norm_act: groups=%d must divide channels=%d",
                p->groups, p->channels);
  if (p->channels >= (1 << 24))
    return fail(BEVK_ERR_INDEX_OVERFLOW, "group_norm_act: %d channels (below 2^24)", p->channels);
  if (p->act != BEVK_ACT_NONE && p->act != BEVK_ACT_RELU && p->act != BEVK_ACT_SILU)
    return fail(BEVK_ERR_UNSUPPORTED, "group_norm_act: activation %d", p->act);
  if (!(p->eps >= 0.f) || std::isinf(p->eps))
    return fail(BEVK_ERR_INVALID_ARGUMENT, "group_norm_act: eps must be finite and >= 0");
  if (p->pixels >= (int64_t(1) << 31) - (1 << 20))
    return fail(BEVK_ERR_INDEX_OVERFLOW, "group_norm_act: %lld pixels exceed 31-bit indexing",
                static_cast<long long>(p->pixels));
  if (static_cast<int64_t>(p->batch) * p->channels >= int64_t(1) << 31)
    return fail(BEVK_ERR_INDEX_OVERFLOW, "group_norm_act: batch x channels exceed 31-bit indexing");
  for (int i = 0; i < 2; ++i)
    if (p->input_strides[i] < 0 || p->output_strides[i] < 0 ||
        (backward && p->grad_output_strides[i] < 0))
      return fail(BEVK_ERR_INVALID_ARGUMENT, "group_norm_act: negative strides");
  return BEVK_OK;
}

// Checks the arguments of the embedding gradient (not its pointers).
int check_embedding_backward(const bevk_embedding_backward_args *a) {
  if (!a) return fail(BEVK_ERR_INVALID_ARGUMENT, "embedding_backward: null arguments");
  if (!known_dtype(a->grad_output_dtype) ||
      (a->grad_table_dtype != a->grad_output_dtype && a->grad_table_dtype != BEVK_DTYPE_F32))
    return fail(BEVK_ERR_UNSUPPORTED,
                "embedding_backward: dtypes %d -> %d (f32, f16, bf16, into the same or f32)",
                a->grad_output_dtype, a->grad_table_dtype);
  if (a->num_ids < 0 || a->num_rows < 0 || a->dim <= 0)
    return fail(BEVK_ERR_INVALID_ARGUMENT, "embedding_backward: bad sizes");
  if (a->grad_output_ld < 0 || a->grad_table_ld < a->dim)
    return fail(BEVK_ERR_INVALID_ARGUMENT, "embedding_backward: bad row strides");
  if (a->num_ids >= (int64_t(1) << 31) - (1 << 16) || a->num_rows >= (int64_t(1) << 31) - 1 ||
      a->dim >= (1 << 24))
    return fail(BEVK_ERR_INDEX_OVERFLOW,
                "embedding_backward: ids and rows are indexed in 31 bits, columns in 24");
  return BEVK_OK;
}

cudaStream_t cuda_stream(bevk_stream_t s) { return reinterpret_cast<cudaStream_t>(s); }

int zero(void *p, size_t bytes, cudaStream_t stream, const char *what) {
  if (p == nullptr || bytes == 0) return BEVK_OK;
  return launched(cudaMemsetAsync(p, 0, bytes, stream), what);
}

}  // namespace

extern "C" {

BEVK_API size_t bevk_group_norm_act_workspace_bytes(const bevk_group_norm_problem *p,
                                                    int backward) {
  clear_error();
  if (check_group_norm(p, backward != 0) != BEVK_OK) return 0;
  if (p->batch == 0 || p->pixels == 0) return 0;
  return group_norm_workspace_bytes(p, backward != 0);
}

BEVK_API int bevk_group_norm_act_forward(const bevk_group_norm_problem *p, const void *input,
                                         const void *weight, const void *bias, void *output,
                                         float *mean, float *rstd, void *workspace,
                                         size_t workspace_bytes, bevk_stream_t stream) {
  clear_error();
  const int st = check_group_norm(p, false);
  if (st != BEVK_OK) return st;
  if ((mean == nullptr) != (rstd == nullptr))
    return fail(BEVK_ERR_INVALID_ARGUMENT, "group_norm_act_forward: mean and rstd go together");
  if (p->batch == 0) return BEVK_OK;
  if (p->pixels == 0) {
    const size_t n = sizeof(float) * static_cast<size_t>(p->batch) * p->groups;
    const int s = zero(mean, n, cuda_stream(stream), "group_norm_act_forward");
    return s != BEVK_OK ? s : zero(rstd, n, cuda_stream(stream), "group_norm_act_forward");
  }
  if (!input || !output || !workspace)
    return fail(BEVK_ERR_INVALID_ARGUMENT, "group_norm_act_forward: null pointer");
  if (!aligned(workspace, 16))
    return fail(BEVK_ERR_MISALIGNED, "group_norm_act_forward: workspace must be 16-byte aligned");
  return launch_group_norm_forward(p, input, weight, bias, output, mean, rstd, workspace,
                                   workspace_bytes, cuda_stream(stream));
}

BEVK_API int bevk_group_norm_act_backward(const bevk_group_norm_problem *p,
                                          const void *grad_output, const void *input,
                                          const float *mean, const float *rstd,
                                          const void *weight, const void *bias,
                                          void *grad_input, void *grad_weight, void *grad_bias,
                                          void *workspace, size_t workspace_bytes,
                                          bevk_stream_t stream) {
  clear_error();
  const int st = check_group_norm(p, true);
  if (st != BEVK_OK) return st;
  if (!grad_input && !grad_weight && !grad_bias) return BEVK_OK;
  if (p->batch == 0 || p->pixels == 0) {
    const size_t n = dtype_size(p->param_dtype) * static_cast<size_t>(p->channels);
    const int s = zero(grad_weight, n, cuda_stream(stream), "group_norm_act_backward");
    return s != BEVK_OK ? s : zero(grad_bias, n, cuda_stream(stream), "group_norm_act_backward");
  }
  if (!grad_output || !input || !mean || !rstd || !workspace)
    return fail(BEVK_ERR_INVALID_ARGUMENT, "group_norm_act_backward: null pointer");
  if (!aligned(workspace, 16))
    return fail(BEVK_ERR_MISALIGNED, "group_norm_act_backward: workspace must be 16-byte aligned");
  return launch_group_norm_backward(p, grad_output, input, mean, rstd, weight, bias, grad_input,
                                    grad_weight, grad_bias, workspace, workspace_bytes,
                                    cuda_stream(stream));
}

BEVK_API int bevk_embedding_forward(const void *table, int64_t table_ld, const void *ids,
                                    int ids_are_64bit, int64_t num_ids, int64_t num_rows,
                                    int dim, float scale, void *output, int dtype,
                                    bevk_stream_t stream) {
  clear_error();
  if (!known_dtype(dtype))
    return fail(BEVK_ERR_UNSUPPORTED, "embedding_forward: dtype %d (f32, f16, bf16)", dtype);
  if (num_ids < 0 || num_rows < 0 || dim <= 0 || table_ld < 0)
    return fail(BEVK_ERR_INVALID_ARGUMENT, "embedding_forward: bad sizes");
  if (dim >= (1 << 24))
    return fail(BEVK_ERR_INDEX_OVERFLOW, "embedding_forward: %d columns (below 2^24)", dim);
  if (num_ids == 0) return BEVK_OK;
  if (!ids || !output || (!table && num_rows > 0))
    return fail(BEVK_ERR_INVALID_ARGUMENT, "embedding_forward: null pointer");
  return launch_embedding_forward(table, table_ld, ids, ids_are_64bit != 0, num_ids, num_rows, dim,
                                  scale, output, dtype, cuda_stream(stream));
}

BEVK_API size_t bevk_embedding_backward_workspace_bytes(const bevk_embedding_backward_args *a) {
  clear_error();
  if (check_embedding_backward(a) != BEVK_OK || a->num_ids == 0 || a->num_rows == 0) return 0;
  return embedding_backward_workspace_bytes(a);
}

BEVK_API int bevk_embedding_backward(const bevk_embedding_backward_args *a,
                                     const void *grad_output, const void *ids, void *grad_table,
                                     void *workspace, size_t workspace_bytes,
                                     bevk_stream_t stream) {
  clear_error();
  const int st = check_embedding_backward(a);
  if (st != BEVK_OK) return st;
  if (a->num_rows == 0) return BEVK_OK;
  if (!grad_table) return fail(BEVK_ERR_INVALID_ARGUMENT, "embedding_backward: null pointer");
  if (a->num_ids == 0) {
    if (a->accumulate) return BEVK_OK;
    const size_t size = dtype_size(a->grad_table_dtype);
    return launched(cudaMemset2DAsync(grad_table, a->grad_table_ld * size, 0, a->dim * size,
                                      a->num_rows, cuda_stream(stream)),
                    "embedding_backward");
  }
  if (!grad_output || !ids)
    return fail(BEVK_ERR_INVALID_ARGUMENT, "embedding_backward: null pointer");
  const size_t need = embedding_backward_workspace_bytes(a);
  if (!workspace || workspace_bytes < need)
    return fail(BEVK_ERR_WORKSPACE, "embedding_backward: workspace of %zu bytes, needs %zu",
                workspace_bytes, need);
  if (!aligned(workspace, 256))
    return fail(BEVK_ERR_MISALIGNED, "embedding_backward: workspace must be 256-byte aligned");
  return launch_embedding_backward(a, grad_output, ids, grad_table, workspace,
                                   cuda_stream(stream));
}

BEVK_API size_t bevk_grad_clip_workspace_bytes(int num_tensors) {
  clear_error();
  return num_tensors < 0 ? 0 : grad_clip_workspace_bytes(num_tensors);
}

BEVK_API int bevk_grad_clip(const bevk_grad_tensor *tensors, int num_tensors, int norm_kind,
                            float max_norm, float eps, int scale, float *norm_out,
                            void *workspace, size_t workspace_bytes, bevk_stream_t stream) {
  clear_error();
  if (num_tensors < 0 || (num_tensors > 0 && !tensors) || !norm_out)
    return fail(BEVK_ERR_INVALID_ARGUMENT, "grad_clip: null pointer or negative count");
  if (norm_kind != BEVK_NORM_L2 && norm_kind != BEVK_NORM_INF)
    return fail(BEVK_ERR_UNSUPPORTED, "grad_clip: norm kind %d", norm_kind);
  if (scale && (!(max_norm >= 0.f) || !(eps >= 0.f)))
    return fail(BEVK_ERR_INVALID_ARGUMENT, "grad_clip: max_norm and eps must be >= 0");
  int64_t total = 0;
  for (int i = 0; i < num_tensors; ++i) {
    const bevk_grad_tensor &t = tensors[i];
    if (t.numel < 0) return fail(BEVK_ERR_INVALID_ARGUMENT, "grad_clip: tensor %d: numel", i);
    if (!known_dtype(t.grad_dtype) || (scale && !known_dtype(t.out_dtype)))
      return fail(BEVK_ERR_UNSUPPORTED, "grad_clip: tensor %d: dtype (f32, f16, bf16)", i);
    if (t.numel == 0) continue;
    if (!t.grad || (scale && !t.out))
      return fail(BEVK_ERR_INVALID_ARGUMENT, "grad_clip: tensor %d: null pointer", i);
    if (!aligned(t.grad, dtype_size(t.grad_dtype)) ||
        (scale && !aligned(t.out, dtype_size(t.out_dtype))))
      return fail(BEVK_ERR_MISALIGNED, "grad_clip: tensor %d: not aligned to its type", i);
    if (scale && t.grad == t.out && t.grad_dtype != t.out_dtype)
      return fail(BEVK_ERR_INVALID_ARGUMENT, "grad_clip: tensor %d: in place with two types", i);
    total += t.numel;
  }
  if (total == 0) return zero(norm_out, sizeof(float), cuda_stream(stream), "grad_clip");
  if (!workspace || workspace_bytes < grad_clip_workspace_bytes(num_tensors))
    return fail(BEVK_ERR_WORKSPACE, "grad_clip: workspace of %zu bytes, needs %zu",
                workspace_bytes, grad_clip_workspace_bytes(num_tensors));
  if (!aligned(workspace, 16))
    return fail(BEVK_ERR_MISALIGNED, "grad_clip: workspace must be 16-byte aligned");
  return launch_grad_clip(tensors, num_tensors, norm_kind, max_norm, eps, scale, norm_out,
                          workspace, cuda_stream(stream));
}

}  // extern "C"
