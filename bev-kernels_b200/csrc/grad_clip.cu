// grad_clip.cu -- the global norm of many gradient tensors and clipping by it.
//
//   norm = sqrt(sum_t sum_i g^2)  or  max |g|
//   c = min(1, max_norm / (norm + eps)),  out = c g
//
// The norm has to be known before the first element is scaled, so the data is
// swept twice: once for the norm, once to scale (not at all where it would be
// scaled in place by 1).  HBM carries one read for the norm, and the scaled
// copy's read and write, less what the second sweep still finds in L2: it
// runs over the tiles in the opposite order.  One cooperative launch does
// both sweeps for up to 1000 tensors, whose addresses travel as kernel
// parameters -- nothing is copied to the device first.
//
// The tensors are cut into tiles of one size (a tensor's last one is shorter)
// and every CTA takes a contiguous run of tiles.  Squares are summed in fp32
// within a tile and thread (in fp64 where they leave its range), and those sums in
// fp64 in a fixed order.
//
// Bound by memory: 68 M bf16 elements clipped into fp32 take 97 us on the device
// (136 MB read twice, 272 MB written: 5.6 TB/s), 28 us of it the norm, whose rate
// grows from 4.8 TB/s at this size to 7.2 at 4 GB.  40 tensors of 1.3 M elements
// within the limit take 6 us: launch, one round trip to memory, the grid's
// meeting.  Keeping 192 KB a CTA pair in flight through asynchronous copies that
// run on across tiles measured 109 us.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <new>
#include <vector>

#include "bevk_internal.h"
#include "vec_io.cuh"

namespace cg = cooperative_groups;

namespace bevk {
namespace {

// Two CTAs of 512 threads with four vectors each in flight.  Batches of 8, 1 or
// 3 to 4 CTAs per SM, and CTAs of 256 or 1024 threads measured the same or slower
// (norm and scaled copy of 68 M bf16 elements into fp32: 101 us; 105 to 119).
constexpr int kThreads = 512;
constexpr int kCtasPerSm = 2;
constexpr int kBatch = 4;
constexpr int kMostTile = 32768;  // elements
constexpr int kMostTensors = 1000;  // of one launch: 32 KB of kernel parameters hold them
constexpr int kFewTensors = 100;    // fit the first 4 KB of parameters
constexpr int kMostCtas = 148 * 4;

enum Mode { kBoth = 0, kNormOnly = 1, kScaleOnly = 2 };

template <int MOST>
struct ClipParams {
  const void *in[MOST];
  void *out[MOST];
  int64_t numel[MOST];
  int first_tile[MOST + 1];
  unsigned char types[MOST];  // grad dtype + 4 * out dtype
  int tensors, tiles, tile;   // tile: elements, a multiple of 8
  int mode, inf_norm, scale;
  int partials;               // partial results that make up the norm
  float max_norm, eps;
  float *norm_out;            // null: another launch writes it
  double *partial;            // this launch's in the norm sweep, all in the other
};
static_assert(sizeof(ClipParams<kFewTensors>) <= 4096, "parameter space");
static_assert(sizeof(ClipParams<kMostTensors>) <= 32764, "parameter space");

// max that keeps a NaN
template <typename F>
__device__ __forceinline__ F max_nan(F m, F v) {
  return (v > m || v != v) ? v : m;
}

// Four running results, so that consecutive elements do not wait for one another.
template <bool INF>
struct Sum {
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  __device__ __forceinline__ void take(int i, float v) {
    acc[i & 3] = INF ? max_nan(acc[i & 3], fabsf(v)) : fmaf(v, v, acc[i & 3]);
  }
  __device__ __forceinline__ float value() const {
    if (INF) return max_nan(max_nan(acc[0], acc[1]), max_nan(acc[2], acc[3]));
    return (acc[0] + acc[1]) + (acc[2] + acc[3]);
  }
};

// Elements before p's first boundary of `bytes` (at most n).
template <typename T>
__device__ __forceinline__ int head_of(const T *p, int n, int bytes) {
  const int off = static_cast<int>(reinterpret_cast<uintptr_t>(p) & (bytes - 1));
  return min(n, off ? (bytes - off) / static_cast<int>(sizeof(T)) : 0);
}

// A thread's squares of a tile in fp64, for those that leave fp32's range: the same
// elements as below.
template <typename T>
__device__ __noinline__ double wide_squares(const T *p, int n) {
  constexpr int V = vio::Full<T>::value;
  const int tid = threadIdx.x, head = head_of(p, n, 16);
  double sum = 0.0;
  const auto take = [&](T e) {
    const double v = vio::widen(e);
    sum = fma(v, v, sum);
  };
  if (tid < head) take(p[tid]);
  const T *body = p + head;
  const int vecs = (n - head) / V;
  for (int i = tid; i < vecs; i += kThreads)
    for (int e = 0; e < V; ++e) take(body[i * V + e]);
  if (tid < n - head - vecs * V) take(body[vecs * V + tid]);
  return sum;
}

// Squares are summed in fp32, which holds them to its precision while the result
// is not below 2^-100 (what is lost of subnormal squares is 2^-144 at most) and
// does not overflow; else, except where all elements are zero, once more in fp64.
constexpr float kLeastSquares = 0x1p-100f, kMostSquares = 0x1.fffffep127f;

template <typename T, bool INF>
__device__ __forceinline__ double norm_tile(const T *p, int n) {
  constexpr int V = vio::Full<T>::value, B = kBatch;
  Sum<INF> s;
  unsigned bits = 0;  // whether any element is not zero
  const int tid = threadIdx.x, head = head_of(p, n, 16);
  const auto take_one = [&](int k, T e) {
    const float v = vio::widen(e);
    s.take(k, v);
    bits |= __float_as_uint(fabsf(v));
  };
  if (tid < head) take_one(0, p[tid]);
  const T *body = p + head;
  const int vecs = (n - head) / V;
  const auto take = [&](const vio::Pack<T, V> &q) {
    float f[V];
    vio::unpack(q, f);
#pragma unroll
    for (int e = 0; e < V; ++e) s.take(e, f[e]);
    if (!INF) bits |= (q.w[0] | q.w[1] | q.w[2] | q.w[3]) & (sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu);
  };
  int i = tid;
  for (; i + (B - 1) * kThreads < vecs; i += B * kThreads) {
    vio::Pack<T, V> q[B];
#pragma unroll
    for (int k = 0; k < B; ++k) q[k] = vio::load_pack<T, V>(body + (i + k * kThreads) * V);
#pragma unroll
    for (int k = 0; k < B; ++k) take(q[k]);
  }
  for (; i < vecs; i += kThreads) take(vio::load_pack<T, V>(body + i * V));
  const int tail = n - head - vecs * V;
  if (tid < tail) take_one(1, body[vecs * V + tid]);
  const float v = s.value();
  if (!INF && ((v < kLeastSquares && bits != 0) || !(v <= kMostSquares))) return wide_squares(p, n);
  return v;
}

// Scales one tile.  A thread takes as many elements at a time as make 16 bytes
// of the wider type, so that the warp's accesses to both sides are contiguous.
template <typename T, typename To>
__device__ __forceinline__ void scale_tile(const T *p, To *o, int n, float c) {
  constexpr int V = 16 / (sizeof(T) > sizeof(To) ? sizeof(T) : sizeof(To)), B = kBatch;
  const int tid = threadIdx.x, head = head_of(p, n, V * sizeof(T));
  if (tid < head) o[tid] = vio::narrow<To>(c * vio::widen(p[tid]));
  const T *body = p + head;
  To *dst = o + head;
  const int vecs = (n - head) / V;
  const bool vector = reinterpret_cast<uintptr_t>(dst) % (V * sizeof(To)) == 0;
  const auto put = [&](const vio::Pack<T, V> &q, int i) {
    float f[V];
    vio::unpack(q, f);
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] *= c;
    if (vector) {
      vio::store_pack_streaming<To, V>(dst + i * V, vio::pack<To, V>(f));
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) dst[i * V + e] = vio::narrow<To>(f[e]);
    }
  };
  int i = tid;
  for (; i + (B - 1) * kThreads < vecs; i += B * kThreads) {
    vio::Pack<T, V> q[B];
#pragma unroll
    for (int k = 0; k < B; ++k) q[k] = vio::load_pack<T, V>(body + (i + k * kThreads) * V);
#pragma unroll
    for (int k = 0; k < B; ++k) put(q[k], i + k * kThreads);
  }
  for (; i < vecs; i += kThreads) put(vio::load_pack<T, V>(body + i * V), i);
  const int tail = n - head - vecs * V;
  if (tid < tail) {
    const int i = vecs * V + tid;
    dst[i] = vio::narrow<To>(c * vio::widen(body[i]));
  }
}

template <typename T>
__device__ __forceinline__ void scale_any(const void *in, void *out, int64_t at, int n,
                                          int out_dtype, float c) {
  const T *p = static_cast<const T *>(in) + at;
  switch (out_dtype) {
    case BEVK_DTYPE_F16: scale_tile(p, static_cast<__half *>(out) + at, n, c); break;
    case BEVK_DTYPE_BF16: scale_tile(p, static_cast<__nv_bfloat16 *>(out) + at, n, c); break;
    default: scale_tile(p, static_cast<float *>(out) + at, n, c);
  }
}

// Sum (or max) of one double per thread over the CTA, in a fixed order; every
// thread gets it.
__device__ double cta_reduce(double v, bool inf_norm, double *s_part) {
  __syncthreads();
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) {
    const double u = __shfl_xor_sync(0xffffffffu, v, m);
    v = inf_norm ? max_nan(v, u) : v + u;
  }
  if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = v;
  __syncthreads();
  constexpr int kWarps = kThreads / 32;
  v = s_part[threadIdx.x & (kWarps - 1)];
#pragma unroll
  for (int m = kWarps / 2; m > 0; m >>= 1) {
    const double u = __shfl_xor_sync(0xffffffffu, v, m);
    v = inf_norm ? max_nan(v, u) : v + u;
  }
  return v;
}

template <typename T>
__device__ __forceinline__ double norm_any(const void *p, int64_t at, int n, bool inf_norm) {
  const T *q = static_cast<const T *>(p) + at;
  return inf_norm ? norm_tile<T, true>(q, n) : norm_tile<T, false>(q, n);
}

template <int MOST>
__global__ void __launch_bounds__(kThreads, kCtasPerSm)
    grad_clip_kernel(const __grid_constant__ ClipParams<MOST> p) {
  __shared__ double s_part[kThreads / 32];
  const bool inf_norm = p.inf_norm != 0;
  const int t0 = static_cast<int>(static_cast<int64_t>(p.tiles) * blockIdx.x / gridDim.x);
  const int t1 = static_cast<int>(static_cast<int64_t>(p.tiles) * (blockIdx.x + 1) / gridDim.x);
  // the tensor that tile t0 lies in
  int k = 0;
  for (int hi = p.tensors; hi - k > 1;) {
    const int mid = (k + hi) >> 1;
    if (p.first_tile[mid] <= t0) k = mid;
    else hi = mid;
  }

  if (p.mode != kScaleOnly) {
    double sum = 0.0;
    for (int t = t0; t < t1; ++t) {
      while (t >= p.first_tile[k + 1]) ++k;
      const int64_t at = static_cast<int64_t>(t - p.first_tile[k]) * p.tile;
      const int n = static_cast<int>(min(static_cast<int64_t>(p.tile), p.numel[k] - at));
      double v;
      switch (p.types[k] & 3) {
        case BEVK_DTYPE_F16: v = norm_any<__half>(p.in[k], at, n, inf_norm); break;
        case BEVK_DTYPE_BF16: v = norm_any<__nv_bfloat16>(p.in[k], at, n, inf_norm); break;
        default: v = norm_any<float>(p.in[k], at, n, inf_norm);
      }
      sum = inf_norm ? max_nan(sum, v) : sum + v;
    }
    sum = cta_reduce(sum, inf_norm, s_part);
    if (threadIdx.x == 0) __stcg(p.partial + blockIdx.x, sum);
    if (p.mode == kNormOnly) return;
    cg::this_grid().sync();
  }

  double total = 0.0;
  for (int i = threadIdx.x; i < p.partials; i += kThreads) {
    const double v = __ldcg(p.partial + i);
    total = inf_norm ? max_nan(total, v) : total + v;
  }
  total = cta_reduce(total, inf_norm, s_part);
  const float norm = static_cast<float>(inf_norm ? total : sqrt(total));
  if (p.norm_out != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *p.norm_out = norm;
  if (!p.scale) return;
  float c = p.max_norm / (norm + p.eps);
  if (c > 1.f) c = 1.f;  // a NaN stays
  while (k + 1 < p.tensors && p.first_tile[k + 1] < t1) ++k;  // where the norm sweep ends
  for (int t = t1 - 1; t >= t0; --t) {
    while (t < p.first_tile[k]) --k;
    if (c == 1.f && p.in[k] == p.out[k]) continue;
    const int64_t at = static_cast<int64_t>(t - p.first_tile[k]) * p.tile;
    const int n = static_cast<int>(min(static_cast<int64_t>(p.tile), p.numel[k] - at));
    const int out_dtype = p.types[k] >> 2;
    switch (p.types[k] & 3) {
      case BEVK_DTYPE_F16: scale_any<__half>(p.in[k], p.out[k], at, n, out_dtype, c); break;
      case BEVK_DTYPE_BF16: scale_any<__nv_bfloat16>(p.in[k], p.out[k], at, n, out_dtype, c); break;
      default: scale_any<float>(p.in[k], p.out[k], at, n, out_dtype, c);
    }
  }
}

template <int MOST>
int resident_ctas() {
  static thread_local int seen_device = -1, seen_ctas = 0;
  const int dev = current_device();
  if (dev < 0) return 0;
  if (seen_device == dev) return seen_ctas;
  int per_sm = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, grad_clip_kernel<MOST>, kThreads, 0) !=
      cudaSuccess)
    return 0;
  seen_device = dev;
  seen_ctas = std::min(kMostCtas, per_sm * device_info(dev).sm_count);
  return seen_ctas;
}

struct Call {
  int inf_norm, scale;
  float max_norm, eps;
  float *norm_out;
  double *partial;
};

// One launch over tensors[0, n).  In kNormOnly mode `base` is where this
// launch's partials begin and *partials counts them up; in kScaleOnly mode
// *partials is their number.
template <int MOST>
int launch(const bevk_grad_tensor *tensors, int n, const Call &c, Mode mode, int *partials,
           bool write_norm, cudaStream_t stream) {
  const int ctas = resident_ctas<MOST>();
  if (ctas <= 0) return fail(BEVK_ERR_CUDA, "grad_clip: occupancy query failed");
  static thread_local ClipParams<MOST> p;
  int64_t total = 0;
  for (int i = 0; i < n; ++i) total += tensors[i].numel;
  // a tile a CTA where there is little (each costs a round trip to memory), of
  // 2048 to 32768 elements
  int64_t tile = (total / ctas + 2047) / 2048 * 2048;
  tile = std::max<int64_t>(2048, std::min<int64_t>(kMostTile, tile));
  int64_t tiles = 0;
  p.tensors = 0;
  for (int i = 0; i < n; ++i) {
    if (tensors[i].numel == 0) continue;
    const int k = p.tensors++;
    p.in[k] = tensors[i].grad;
    p.out[k] = c.scale ? tensors[i].out : const_cast<void *>(tensors[i].grad);
    p.numel[k] = tensors[i].numel;
    p.types[k] = static_cast<unsigned char>(tensors[i].grad_dtype +
                                            4 * (c.scale ? tensors[i].out_dtype : 0));
    p.first_tile[k] = static_cast<int>(tiles);
    tiles += (tensors[i].numel + tile - 1) / tile;
    if (tiles >= (int64_t(1) << 31) - 1)
      return fail(BEVK_ERR_INDEX_OVERFLOW, "grad_clip: too many elements");
  }
  p.first_tile[p.tensors] = static_cast<int>(tiles);
  p.tiles = static_cast<int>(tiles);
  p.tile = static_cast<int>(tile);
  p.mode = mode;
  p.inf_norm = c.inf_norm;
  p.scale = c.scale;
  p.max_norm = c.max_norm;
  p.eps = c.eps;
  p.norm_out = write_norm ? c.norm_out : nullptr;
  p.partial = c.partial + (mode == kNormOnly ? *partials : 0);
  const int grid = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(ctas, tiles)));
  if (mode == kNormOnly) *partials += grid;
  p.partials = mode == kBoth ? grid : *partials;
  if (mode == kBoth) {
    void *args[] = {&p};
    return launched(
        cudaLaunchCooperativeKernel(reinterpret_cast<void *>(grad_clip_kernel<MOST>), dim3(grid),
                                    dim3(kThreads), args, 0, stream),
        "grad_clip_kernel");
  }
  grad_clip_kernel<MOST><<<grid, kThreads, 0, stream>>>(p);
  return check_launch("grad_clip_kernel");
}

int chunks_of(int tensors) { return std::max(1, (tensors + kMostTensors - 1) / kMostTensors); }

// Outputs are disjoint from one another and from every gradient but their own.
// Two lists, since tensors of one buffer mostly come in order and then nothing
// has to be sorted.
int check_overlap(const bevk_grad_tensor *t, int n) {
  struct Span {
    uintptr_t begin, end;
    int tensor;
  };
  std::vector<Span> outs, grads;  // a gradient scaled in place is an output only
  outs.reserve(static_cast<size_t>(n));
  grads.reserve(static_cast<size_t>(n));
  for (int i = 0; i < n; ++i) {
    if (t[i].numel == 0) continue;
    const auto a = reinterpret_cast<uintptr_t>(t[i].out);
    const auto b = reinterpret_cast<uintptr_t>(t[i].grad);
    outs.push_back({a, a + t[i].numel * dtype_size(t[i].out_dtype), i});
    if (t[i].grad != t[i].out)
      grads.push_back({b, b + t[i].numel * dtype_size(t[i].grad_dtype), i});
  }
  const auto less = [](const Span &x, const Span &y) { return x.begin < y.begin; };
  for (std::vector<Span> *v : {&outs, &grads})
    if (!std::is_sorted(v->begin(), v->end(), less)) std::sort(v->begin(), v->end(), less);
  // in order of address over both: no output before the end of anything, no
  // gradient before the end of an output
  uintptr_t out_end = 0, grad_end = 0;
  size_t i = 0, j = 0;
  while (i < outs.size() || j < grads.size()) {
    const bool out = j == grads.size() || (i < outs.size() && outs[i].begin <= grads[j].begin);
    const Span &s = out ? outs[i++] : grads[j++];
    if (s.begin < out_end || (out && s.begin < grad_end))
      return fail(BEVK_ERR_INVALID_ARGUMENT,
                  "grad_clip: tensor %d overlaps another tensor that is written or read", s.tensor);
    uintptr_t &end = out ? out_end : grad_end;
    end = std::max(end, s.end);
  }
  return BEVK_OK;
}

}  // namespace

size_t grad_clip_workspace_bytes(int tensors) {
  return sizeof(double) * kMostCtas * static_cast<size_t>(chunks_of(tensors));
}

int launch_grad_clip(const bevk_grad_tensor *tensors, int n, int norm_kind, float max_norm,
                     float eps, int scale, float *norm_out, void *ws, cudaStream_t stream) {
  if (scale) {
    try {
      const int st = check_overlap(tensors, n);
      if (st != BEVK_OK) return st;
    } catch (const std::bad_alloc &) {
      return fail(BEVK_ERR_INVALID_ARGUMENT, "grad_clip: out of host memory");
    }
  }
  const Call c = {norm_kind == BEVK_NORM_INF, scale, max_norm, eps, norm_out,
                  static_cast<double *>(ws)};
  int partials = 0;
  if (n <= kFewTensors) return launch<kFewTensors>(tensors, n, c, kBoth, &partials, true, stream);
  if (n <= kMostTensors) return launch<kMostTensors>(tensors, n, c, kBoth, &partials, true, stream);
  // more tensors than one launch's parameters hold: the norms first, then the
  // scaling, a launch per 1000 tensors each
  for (int mode : {kNormOnly, kScaleOnly}) {
    for (int i = 0; i < n; i += kMostTensors) {
      if (mode == kScaleOnly && !scale && i > 0) break;  // the first one wrote the norm
      const int st = launch<kMostTensors>(tensors + i, std::min(kMostTensors, n - i), c,
                                          static_cast<Mode>(mode), &partials, i == 0, stream);
      if (st != BEVK_OK) return st;
    }
  }
  return BEVK_OK;
}

}  // namespace bevk
