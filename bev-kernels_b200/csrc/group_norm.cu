// group_norm.cu -- group norm with a fused activation on channels-last
// tensors, forward and backward.
//
// Mathematics, per image n and group g of K = C/G channels over HW pixels
// (m = K * HW values):
//   forward   mu = mean(x), r = 1 / sqrt(var + eps),
//             z = w_c (x - mu) r + b_c,  y = act(z)
//   backward  dz = dy act'(z),  db_c = sum dz,  dw_c = sum dz xhat,
//             xhat = (x - mu) r,
//             dx = r (w_c dz - (s1 + xhat s2) / m),
//             s1 = sum_group w_c dz,  s2 = sum_group w_c dz xhat.
//
// Both directions are two sweeps over the same data with a reduction between
// them: 2 (forward) or 3 (backward) passes over the tensor are what HBM has
// to carry, so they are bound by memory once the tensors are large and by the
// launch and the reduction's latency when they are small.  One cooperative
// launch does both sweeps.  Every CTA owns a slab of pixels of one image (all
// channels where C allows): consecutive threads take consecutive 16-byte
// channel vectors, so a warp reads whole lines, and a thread keeps the same
// channels for the whole slab (its weights stay in registers).  After the
// first sweep each CTA leaves one partial result per group, the grid meets,
// and each CTA merges the partials of its own images in a fixed order before
// its second sweep.  Images are taken in waves small enough that the second
// sweep finds the wave in L2.
//
// The variance is not a difference of sums of squares: each thread takes mean
// and squared deviations of a few pixels at a time in registers, and such
// (count, mean, M2) triples are merged pairwise all the way up, which holds
// when the mean is far from zero and when single values are far out.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "bevk_internal.h"
#include "vec_io.cuh"

namespace cg = cooperative_groups;

namespace bevk {
namespace {

constexpr int kThreads = 512;
constexpr int kBatch = 4;  // pixels a thread loads before it uses them

// Waves: both sweeps' tensors of one wave of images stay below this, a good
// half of the 126 MB L2.
constexpr int64_t kWaveBytes = int64_t(72) << 20;

struct GnParams {
  const void *x, *dy, *w, *b;
  void *out;           // y, or dx
  void *dw, *db;
  float *mean, *rstd;  // written by the forward, read by the backward
  float2 *gpart;       // [(image * nb + block) * Gb + group][S]
  float2 *cpart;       // [cta][channels of its block] (backward)
  int64_t xs[2], os[2], gs[2];
  int N, C, G, K;      // K = C / G
  int HW;
  int S;               // slabs per image
  int nb;              // channel blocks
  int lanes, R;        // threads across a block's channels, rows of pixels
  int Gb;              // most groups that a channel block touches
  int wave;            // images per wave
  int param_dtype, act;
  float eps;
};

struct Moments {
  float n, mean, m2;
};
__device__ __forceinline__ Moments merge(const Moments &a, const Moments &b) {
  const float n = a.n + b.n;
  const float f = n > 0.f ? b.n / n : 0.f;
  const float d = b.mean - a.mean;
  return {n, a.mean + d * f, a.m2 + b.m2 + d * d * (a.n * f)};
}
__device__ __forceinline__ Moments merge_xor(const Moments &a, int mask) {
  const Moments b = {__shfl_xor_sync(0xffffffffu, a.n, mask),
                     __shfl_xor_sync(0xffffffffu, a.mean, mask),
                     __shfl_xor_sync(0xffffffffu, a.m2, mask)};
  // both lanes of a pair merge in the same order, so they hold equal bits
  const bool low = (threadIdx.x & mask) == 0;
  return merge(low ? a : b, low ? b : a);
}

// sigmoid: the fp32 path pays for the accurate exponential, 16-bit results
// hide the fast one's error (a few ulp of fp32) behind their rounding.
template <typename T>
__device__ __forceinline__ float sigmoid(float z) {
  if constexpr (sizeof(T) == 4) return 1.f / (1.f + expf(-z));
  return __fdividef(1.f, 1.f + __expf(-z));
}
template <typename T>
__device__ __forceinline__ float activate(float z, int act) {
  if (act == BEVK_ACT_RELU) return z < 0.f ? 0.f : z;  // NaN stays
  if (act == BEVK_ACT_SILU) return z * sigmoid<T>(z);
  return z;
}
// act'(z); ReLU's is 0 at 0
template <typename T>
__device__ __forceinline__ float slope(float z, int act) {
  if (act == BEVK_ACT_RELU) return z > 0.f ? 1.f : 0.f;
  if (act == BEVK_ACT_SILU) {
    const float s = sigmoid<T>(z);
    return s * (1.f + z * (1.f - s));
  }
  return 1.f;
}

// What a CTA is working on: pixels [p0, p0 + count) of image n.
struct Unit {
  int n, s, p0, count;
};
__device__ __forceinline__ Unit unit_of(const GnParams &p, int64_t u) {
  const int64_t q = u / p.nb;
  Unit t;
  t.n = static_cast<int>(q / p.S);
  t.s = static_cast<int>(q - static_cast<int64_t>(t.n) * p.S);
  t.p0 = static_cast<int>(static_cast<int64_t>(p.HW) * t.s / p.S);
  t.count = static_cast<int>(static_cast<int64_t>(p.HW) * (t.s + 1) / p.S) - t.p0;
  return t;
}
__device__ __forceinline__ int slab_pixels(const GnParams &p, int s) {
  return static_cast<int>(static_cast<int64_t>(p.HW) * (s + 1) / p.S) -
         static_cast<int>(static_cast<int64_t>(p.HW) * s / p.S);
}

// Largest power of two <= 32 of threads per group that lets `groups` groups
// share the CTA.
__device__ __forceinline__ int team_width(int groups) {
  int w = 32;
  while (w > 1 && w * groups > kThreads) w >>= 1;
  return w;
}

// The partials of group g of image n: entry e of [0, count) lies in channel
// block cb0 + e / S, slab e % S.  (A group spans several blocks only where its
// channels do not fit one.)
struct Partials {
  const float2 *base;
  int g, cb0, bw, count;
};
__device__ __forceinline__ Partials partials_of(const GnParams &p, int n, int g, int bw) {
  const int cb0 = g * p.K / bw, cb1 = ((g + 1) * p.K - 1) / bw;
  return {p.gpart + static_cast<int64_t>(n) * p.nb * p.Gb * p.S, g, cb0, bw,
          (cb1 - cb0 + 1) * p.S};
}
__device__ __forceinline__ float2 partial(const GnParams &p, const Partials &q, int e, int *s,
                                          int *channels) {
  const int b = e / p.S, cb = q.cb0 + b;
  *s = e - b * p.S;
  const int c0 = cb * q.bw;
  *channels = min((q.g + 1) * p.K, c0 + q.bw) - max(q.g * p.K, c0);
  return __ldcg(q.base + (static_cast<int64_t>(cb) * p.Gb + (q.g - c0 / p.K)) * p.S + *s);
}

// Mean and rstd of the ng groups from g0 on, from the slabs' partials; the
// threads of a team take the partials in turn.
__device__ void combine_moments(const GnParams &p, int n, int bw, int g0, int ng, float *s_mean,
                                float *s_rstd, bool write) {
  const int w = team_width(ng), j = threadIdx.x & (w - 1);
  for (int base = 0; base < ng; base += kThreads / w) {
    const int gl = base + threadIdx.x / w;
    Moments t = {0.f, 0.f, 0.f};
    if (gl < ng) {
      const Partials q = partials_of(p, n, g0 + gl, bw);
      for (int e = j; e < q.count; e += w) {
        int s, channels;
        const float2 v = partial(p, q, e, &s, &channels);
        t = merge(t, {static_cast<float>(slab_pixels(p, s)) * channels, v.x, v.y});
      }
    }
    for (int m = 1; m < w; m <<= 1) t = merge_xor(t, m);
    if (gl < ng && j == 0) {
      const float rstd = 1.f / sqrtf(t.m2 / t.n + p.eps);
      s_mean[gl] = t.mean;
      s_rstd[gl] = rstd;
      if (write) {
        p.mean[static_cast<int64_t>(n) * p.G + g0 + gl] = t.mean;
        p.rstd[static_cast<int64_t>(n) * p.G + g0 + gl] = rstd;
      }
    }
  }
}

template <typename T, int VEC, bool WHOLE>
__global__ void __launch_bounds__(kThreads) gn_forward_kernel(const __grid_constant__ GnParams p) {
  // statistics columns of a thread: one where its vector lies in one group,
  // else one per channel
  constexpr int NC = WHOLE ? 1 : VEC;
  constexpr int CH = VEC / NC;
  extern __shared__ float s_dyn[];
  float2 *s_red = reinterpret_cast<float2 *>(s_dyn);  // [R][lanes * NC]
  float *s_mean = s_dyn + 2 * kThreads * NC;          // [Gb]
  float *s_rstd = s_mean + p.Gb;
  cg::grid_group grid = cg::this_grid();

  const int tid = threadIdx.x;
  const int r = tid / p.lanes, lane = tid - r * p.lanes;
  const int cb = blockIdx.x % p.nb;
  const int c0 = cb * p.lanes * VEC;
  const int c = c0 + lane * VEC;
  const bool active = r < p.R && c < p.C;
  const int bch = min(p.C - c0, p.lanes * VEC);  // channels of this block
  const int g0 = c0 / p.K, ng = (c0 + bch - 1) / p.K + 1 - g0;
  const T *x = static_cast<const T *>(p.x);
  T *y = static_cast<T *>(p.out);

  for (int n0 = 0; n0 < p.N; n0 += p.wave) {
    const int64_t u0 = static_cast<int64_t>(n0) * p.S * p.nb;
    const int64_t u1 = static_cast<int64_t>(min(p.N, n0 + p.wave)) * p.S * p.nb;
    for (int64_t u = u0 + blockIdx.x; u < u1; u += gridDim.x) {
      const Unit t = unit_of(p, u);
      Moments acc[NC];
#pragma unroll
      for (int k = 0; k < NC; ++k) acc[k] = {0.f, 0.f, 0.f};
      if (active) {
        const T *src = x + t.n * p.xs[0] + t.p0 * p.xs[1] + c;
        int q = r;
        for (; q + (kBatch - 1) * p.R < t.count; q += kBatch * p.R) {
          float v[kBatch][VEC];
#pragma unroll
          for (int i = 0; i < kBatch; ++i)
            vio::unpack(vio::load_pack<T, VEC>(src + static_cast<int64_t>(q + i * p.R) * p.xs[1]),
                        v[i]);
#pragma unroll
          for (int k = 0; k < NC; ++k) {
            float sum = 0.f, m2 = 0.f;
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
#pragma unroll
              for (int e = 0; e < CH; ++e) sum += v[i][k * CH + e];
            const float mean = sum * (1.f / (kBatch * CH));
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
#pragma unroll
              for (int e = 0; e < CH; ++e) {
                const float d = v[i][k * CH + e] - mean;
                m2 += d * d;
              }
            acc[k] = merge(acc[k], {kBatch * CH, mean, m2});
          }
        }
        for (; q < t.count; q += p.R) {
          float v[VEC];
          vio::unpack(vio::load_pack<T, VEC>(src + static_cast<int64_t>(q) * p.xs[1]), v);
#pragma unroll
          for (int k = 0; k < NC; ++k) {
            float sum = 0.f, m2 = 0.f;
#pragma unroll
            for (int e = 0; e < CH; ++e) sum += v[k * CH + e];
            const float mean = sum * (1.f / CH);
#pragma unroll
            for (int e = 0; e < CH; ++e) {
              const float d = v[k * CH + e] - mean;
              m2 += d * d;
            }
            acc[k] = merge(acc[k], {CH, mean, m2});
          }
        }
      }
      const int cols = bch / CH;
      if (active) {
#pragma unroll
        for (int k = 0; k < NC; ++k)
          s_red[r * cols + lane * NC + k] = make_float2(acc[k].mean, acc[k].m2);
      }
      __syncthreads();
      // one team per group merges the rows and columns of the group
      const int w = team_width(ng), j = tid & (w - 1);
      for (int base = 0; base < ng; base += kThreads / w) {
        const int gl = base + tid / w;
        Moments m = {0.f, 0.f, 0.f};
        if (gl < ng) {
          const int k0 = max((g0 + gl) * p.K - c0, 0) / CH;
          const int k1 = min((g0 + gl + 1) * p.K - c0, bch) / CH;
          for (int e = j; e < p.R * (k1 - k0); e += w) {
            const int row = e / (k1 - k0), col = k0 + e - row * (k1 - k0);
            if (row >= t.count) break;
            const float2 v = s_red[row * cols + col];
            m = merge(m, {static_cast<float>((t.count - row + p.R - 1) / p.R * CH), v.x, v.y});
          }
        }
        for (int k = 1; k < w; k <<= 1) m = merge_xor(m, k);
        if (gl < ng && j == 0)
          __stcg(p.gpart + ((static_cast<int64_t>(t.n) * p.nb + cb) * p.Gb + gl) * p.S + t.s,
                 make_float2(m.mean, m.m2));
      }
      __syncthreads();
    }
    grid.sync();
    int have = -1;  // image whose statistics are in shared memory
    for (int64_t u = u0 + blockIdx.x; u < u1; u += gridDim.x) {
      const Unit t = unit_of(p, u);
      if (t.n != have) {
        __syncthreads();
        combine_moments(p, t.n, p.lanes * VEC, g0, ng, s_mean, s_rstd,
                        p.mean != nullptr && t.s == 0);
        have = t.n;
        __syncthreads();
      }
      if (!active) continue;
      float mean[VEC], a[VEC], b[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const int gl = (c + e) / p.K - g0;
        mean[e] = s_mean[gl];
        a[e] = s_rstd[gl] * (p.w ? vio::load_any(p.w, c + e, p.param_dtype) : 1.f);
        b[e] = p.b ? vio::load_any(p.b, c + e, p.param_dtype) : 0.f;
      }
      const T *src = x + t.n * p.xs[0] + t.p0 * p.xs[1] + c;
      T *dst = y + t.n * p.os[0] + t.p0 * p.os[1] + c;
#pragma unroll 4
      for (int q = r; q < t.count; q += p.R) {
        float v[VEC];
        vio::unpack(vio::load_pack<T, VEC>(src + static_cast<int64_t>(q) * p.xs[1]), v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = activate<T>((v[e] - mean[e]) * a[e] + b[e], p.act);
        vio::store<T, VEC>(dst + static_cast<int64_t>(q) * p.os[1], v);
      }
    }
  }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) gn_backward_kernel(const __grid_constant__ GnParams p) {
  extern __shared__ float s_dyn[];
  float2 *s_red = reinterpret_cast<float2 *>(s_dyn);     // [R][lanes * VEC]
  float2 *s_tot = s_red + kThreads * VEC;                // [lanes * VEC] over all units
  float2 *s_sum = s_tot + p.lanes * VEC;                 // [Gb] s1 / m, s2 / m
  cg::grid_group grid = cg::this_grid();

  const int tid = threadIdx.x;
  const int r = tid / p.lanes, lane = tid - r * p.lanes;
  const int cb = blockIdx.x % p.nb;
  const int c0 = cb * p.lanes * VEC;
  const int c = c0 + lane * VEC;
  const bool active = r < p.R && c < p.C;
  const int bch = min(p.C - c0, p.lanes * VEC);
  const int g0 = c0 / p.K, ng = (c0 + bch - 1) / p.K + 1 - g0;
  const float inv_m = 1.f / (static_cast<float>(p.K) * static_cast<float>(p.HW));
  const T *x = static_cast<const T *>(p.x);
  const T *dy = static_cast<const T *>(p.dy);
  T *dx = static_cast<T *>(p.out);

  for (int k = tid; k < p.lanes * VEC; k += kThreads) s_tot[k] = make_float2(0.f, 0.f);
  float w[VEC], b[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    w[e] = active && p.w ? vio::load_any(p.w, c + e, p.param_dtype) : 1.f;
    b[e] = active && p.b ? vio::load_any(p.b, c + e, p.param_dtype) : 0.f;
  }

  for (int n0 = 0; n0 < p.N; n0 += p.wave) {
    const int64_t u0 = static_cast<int64_t>(n0) * p.S * p.nb;
    const int64_t u1 = static_cast<int64_t>(min(p.N, n0 + p.wave)) * p.S * p.nb;
    for (int64_t u = u0 + blockIdx.x; u < u1; u += gridDim.x) {
      const Unit t = unit_of(p, u);
      if (active) {
        float A[VEC], B[VEC], mean[VEC], rstd[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          A[e] = B[e] = 0.f;
          const int64_t g = static_cast<int64_t>(t.n) * p.G + (c + e) / p.K;
          mean[e] = p.mean[g];
          rstd[e] = p.rstd[g];
        }
        const T *px = x + t.n * p.xs[0] + t.p0 * p.xs[1] + c;
        const T *pg = dy + t.n * p.gs[0] + t.p0 * p.gs[1] + c;
#pragma unroll 2
        for (int q = r; q < t.count; q += p.R) {
          float v[VEC], d[VEC];
          vio::unpack(vio::load_pack<T, VEC>(px + static_cast<int64_t>(q) * p.xs[1]), v);
          vio::unpack(vio::load_pack<T, VEC>(pg + static_cast<int64_t>(q) * p.gs[1]), d);
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float xhat = (v[e] - mean[e]) * rstd[e];
            const float dz = d[e] * slope<T>(xhat * w[e] + b[e], p.act);
            A[e] += dz;
            B[e] += dz * xhat;
          }
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) s_red[r * bch + lane * VEC + e] = make_float2(A[e], B[e]);
      }
      __syncthreads();
      // channel sums over the rows; row 0 of s_red becomes w * sum
      for (int k = tid; k < bch; k += kThreads) {
        float2 s = s_red[k];
        for (int row = 1; row < p.R; ++row) {
          const float2 v = s_red[row * bch + k];
          s.x += v.x;
          s.y += v.y;
        }
        s_tot[k].x += s.x;
        s_tot[k].y += s.y;
        const float wk = p.w ? vio::load_any(p.w, c0 + k, p.param_dtype) : 1.f;
        s_red[k] = make_float2(s.x * wk, s.y * wk);
      }
      __syncthreads();
      const int tw = team_width(ng), j = tid & (tw - 1);
      for (int base = 0; base < ng; base += kThreads / tw) {
        const int gl = base + tid / tw;
        float2 s = make_float2(0.f, 0.f);
        if (gl < ng) {
          const int k0 = max((g0 + gl) * p.K - c0, 0), k1 = min((g0 + gl + 1) * p.K - c0, bch);
          for (int k = k0 + j; k < k1; k += tw) {
            s.x += s_red[k].x;
            s.y += s_red[k].y;
          }
        }
        for (int k = 1; k < tw; k <<= 1) {
          s.x += __shfl_xor_sync(0xffffffffu, s.x, k);
          s.y += __shfl_xor_sync(0xffffffffu, s.y, k);
        }
        if (gl < ng && j == 0)
          __stcg(p.gpart + ((static_cast<int64_t>(t.n) * p.nb + cb) * p.Gb + gl) * p.S + t.s, s);
      }
      __syncthreads();
    }
    if (n0 + p.wave >= p.N)
      for (int k = tid; k < bch; k += kThreads)
        __stcg(p.cpart + static_cast<int64_t>(blockIdx.x) * p.lanes * VEC + k, s_tot[k]);
    grid.sync();
    if (p.out != nullptr) {
      int have = -1;
      for (int64_t u = u0 + blockIdx.x; u < u1; u += gridDim.x) {
        const Unit t = unit_of(p, u);
        if (t.n != have) {
          __syncthreads();
          const int tw = team_width(ng), j = tid & (tw - 1);
          for (int base = 0; base < ng; base += kThreads / tw) {
            const int gl = base + tid / tw;
            float2 s = make_float2(0.f, 0.f);
            if (gl < ng) {
              const Partials q = partials_of(p, t.n, g0 + gl, p.lanes * VEC);
              for (int k = j; k < q.count; k += tw) {
                int slab, channels;
                const float2 v = partial(p, q, k, &slab, &channels);
                s.x += v.x;
                s.y += v.y;
              }
            }
            for (int k = 1; k < tw; k <<= 1) {
              s.x += __shfl_xor_sync(0xffffffffu, s.x, k);
              s.y += __shfl_xor_sync(0xffffffffu, s.y, k);
            }
            if (gl < ng && j == 0) s_sum[gl] = make_float2(s.x * inv_m, s.y * inv_m);
          }
          have = t.n;
          __syncthreads();
        }
        if (!active) continue;
        float mean[VEC], rstd[VEC];
        float2 sum[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const int g = (c + e) / p.K;
          mean[e] = p.mean[static_cast<int64_t>(t.n) * p.G + g];
          rstd[e] = p.rstd[static_cast<int64_t>(t.n) * p.G + g];
          sum[e] = s_sum[g - g0];
        }
        const T *px = x + t.n * p.xs[0] + t.p0 * p.xs[1] + c;
        const T *pg = dy + t.n * p.gs[0] + t.p0 * p.gs[1] + c;
        T *dst = dx + t.n * p.os[0] + t.p0 * p.os[1] + c;
#pragma unroll 2
        for (int q = r; q < t.count; q += p.R) {
          float v[VEC], d[VEC];
          vio::unpack(vio::load_pack<T, VEC>(px + static_cast<int64_t>(q) * p.xs[1]), v);
          vio::unpack(vio::load_pack<T, VEC>(pg + static_cast<int64_t>(q) * p.gs[1]), d);
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float xhat = (v[e] - mean[e]) * rstd[e];
            const float dz = d[e] * slope<T>(xhat * w[e] + b[e], p.act);
            v[e] = rstd[e] * (w[e] * dz - (sum[e].x + xhat * sum[e].y));
          }
          vio::store<T, VEC>(dst + static_cast<int64_t>(q) * p.os[1], v);
        }
      }
    }
  }
  // grad_weight and grad_bias: 32 channels at a time, the CTAs' sums in order
  if (p.dw == nullptr && p.db == nullptr) return;
  __syncthreads();
  const int wl = tid & 31, wid = tid >> 5;
  const int bw = p.lanes * VEC;
  for (int base = blockIdx.x * 32; base < p.C; base += gridDim.x * 32) {
    const int ch = base + wl;
    float2 s = make_float2(0.f, 0.f);
    if (ch < p.C) {
      const int blk = ch / bw, k = ch - blk * bw;
      for (int row = blk + wid * p.nb; row < static_cast<int>(gridDim.x);
           row += (kThreads / 32) * p.nb) {
        const float2 v = __ldcg(p.cpart + static_cast<int64_t>(row) * bw + k);
        s.x += v.x;
        s.y += v.y;
      }
    }
    s_red[wid * 32 + wl] = s;
    __syncthreads();
    if (wid == 0 && ch < p.C) {
      for (int k = 1; k < kThreads / 32; ++k) {
        s.x += s_red[k * 32 + wl].x;
        s.y += s_red[k * 32 + wl].y;
      }
      if (p.dw) vio::store_any(p.dw, ch, p.param_dtype, s.y);
      if (p.db) vio::store_any(p.db, ch, p.param_dtype, s.x);
    }
    __syncthreads();
  }
}

// CTAs of `kernel` that are resident at once on the current device (0 on an
// error), remembered per device and shared-memory size.
template <typename K>
int resident_ctas(K kernel, size_t smem) {
  struct Seen {
    int device = -1;
    size_t smem = 0;
    int ctas = 0;
  };
  static thread_local Seen seen;
  const int dev = current_device();
  if (dev < 0) return 0;
  if (seen.device == dev && seen.smem == smem && seen.ctas > 0) return seen.ctas;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           static_cast<int>(smem)) != cudaSuccess)
    return 0;
  int per_sm = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, kThreads, smem) !=
      cudaSuccess)
    return 0;
  seen.device = dev;
  seen.smem = smem;
  seen.ctas = per_sm * device_info(dev).sm_count;
  return seen.ctas;
}

// Channels across the threads of a CTA: everything that follows from the
// shape, the types and the vector width alone.
void set_lanes(GnParams *p, int vec) {
  const int total = p->C / vec;
  p->nb = (total + kThreads - 1) / kThreads;
  p->lanes = (total + p->nb - 1) / p->nb;
  p->nb = (total + p->lanes - 1) / p->lanes;
  p->R = kThreads / p->lanes;
  p->Gb = 0;
  for (int cb = 0; cb < p->nb; ++cb) {
    const int c0 = cb * p->lanes * vec, c1 = std::min(p->C, c0 + p->lanes * vec);
    p->Gb = std::max(p->Gb, (c1 - 1) / p->K + 1 - c0 / p->K);
  }
}

// Waves and slabs for `ctas` resident CTAs; returns the grid.
int set_slabs(GnParams *p, int ctas, int64_t image_bytes) {
  p->wave = static_cast<int>(std::max<int64_t>(
      1, std::min<int64_t>(p->N, kWaveBytes / std::max<int64_t>(image_bytes, 1))));
  const int64_t per_wave = static_cast<int64_t>(p->wave) * p->nb;
  // a slab holds at least a batch of pixels for every thread
  const int64_t most = std::max<int64_t>(1, p->HW / (static_cast<int64_t>(p->R) * kBatch));
  p->S = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(ctas / per_wave, most)));
  const int64_t grid = std::min<int64_t>(per_wave * p->S, ctas);
  return static_cast<int>(std::max<int64_t>(p->nb, grid / p->nb * p->nb));
}

// An upper bound of the CTAs, for the workspace's size: it must not depend on
// the device that the size was asked on.
constexpr int kMostCtas = 148 * 4;

size_t gpart_bytes(const GnParams &p, int S) {
  return sizeof(float2) * static_cast<size_t>(p.N) * p.nb * p.Gb * S;
}

template <typename T, int VEC, bool WHOLE>
int forward(GnParams p, void *ws, size_t ws_bytes, cudaStream_t stream) {
  auto kernel = gn_forward_kernel<T, VEC, WHOLE>;
  const size_t smem = sizeof(float) * (2 * kThreads * (WHOLE ? 1 : VEC) + 2 * p.Gb);
  const int ctas = std::min(kMostCtas, resident_ctas(kernel, smem));
  if (ctas < p.nb) return fail(BEVK_ERR_CUDA, "group_norm_act_forward: occupancy query failed");
  const int grid = set_slabs(&p, ctas, int64_t(2) * p.HW * p.C * sizeof(T));
  if (ws_bytes < gpart_bytes(p, p.S))
    return fail(BEVK_ERR_WORKSPACE, "group_norm_act_forward: workspace of %zu bytes, needs %zu",
                ws_bytes, gpart_bytes(p, p.S));
  p.gpart = static_cast<float2 *>(ws);
  void *args[] = {&p};
  return launched(cudaLaunchCooperativeKernel(reinterpret_cast<void *>(kernel), dim3(grid),
                                              dim3(kThreads), args, smem, stream),
                  "gn_forward_kernel");
}

template <typename T, int VEC>
int backward(GnParams p, void *ws, size_t ws_bytes, cudaStream_t stream) {
  auto kernel = gn_backward_kernel<T, VEC>;
  const size_t bw = static_cast<size_t>(p.lanes) * VEC;
  const size_t smem = sizeof(float2) * (static_cast<size_t>(kThreads) * VEC + bw + p.Gb);
  const int ctas = std::min(kMostCtas, resident_ctas(kernel, smem));
  if (ctas < p.nb) return fail(BEVK_ERR_CUDA, "group_norm_act_backward: occupancy query failed");
  const int grid = set_slabs(&p, ctas, int64_t(3) * p.HW * p.C * sizeof(T));
  const size_t cbytes = sizeof(float2) * bw * grid;
  if (ws_bytes < cbytes + gpart_bytes(p, p.S))
    return fail(BEVK_ERR_WORKSPACE, "group_norm_act_backward: workspace of %zu bytes, needs %zu",
                ws_bytes, cbytes + gpart_bytes(p, p.S));
  p.cpart = static_cast<float2 *>(ws);
  p.gpart = p.cpart + bw * grid;
  void *args[] = {&p};
  return launched(cudaLaunchCooperativeKernel(reinterpret_cast<void *>(kernel), dim3(grid),
                                              dim3(kThreads), args, smem, stream),
                  "gn_backward_kernel");
}

template <typename T>
int dispatch(GnParams &p, bool back, bool vectors, void *ws, size_t ws_bytes,
             cudaStream_t stream) {
  constexpr int V = vio::Full<T>::value;
  if (vectors) {
    set_lanes(&p, V);
    if (back) return backward<T, V>(p, ws, ws_bytes, stream);
    return p.K % V == 0 ? forward<T, V, true>(p, ws, ws_bytes, stream)
                        : forward<T, V, false>(p, ws, ws_bytes, stream);
  }
  set_lanes(&p, 1);
  return back ? backward<T, 1>(p, ws, ws_bytes, stream)
              : forward<T, 1, true>(p, ws, ws_bytes, stream);
}

// 16-byte vectors need every pixel of the tensor on a 16-byte boundary.
bool vector_rows(const void *ptr, const int64_t strides[2], int64_t size) {
  return aligned(ptr, 16) && strides[0] * size % 16 == 0 && strides[1] * size % 16 == 0;
}

GnParams base_params(const bevk_group_norm_problem *q) {
  GnParams p = {};
  for (int i = 0; i < 2; ++i) {
    p.xs[i] = q->input_strides[i];
    p.os[i] = q->output_strides[i];
    p.gs[i] = q->grad_output_strides[i];
  }
  p.N = q->batch;
  p.C = q->channels;
  p.G = q->groups;
  p.K = q->channels / q->groups;
  p.HW = static_cast<int>(q->pixels);
  p.param_dtype = q->param_dtype;
  p.act = q->act;
  p.eps = q->eps;
  return p;
}

}  // namespace

size_t group_norm_workspace_bytes(const bevk_group_norm_problem *q, bool backward) {
  // whichever vector width the call takes
  size_t most = 0;
  const int full = static_cast<int>(16 / dtype_size(q->dtype));
  for (int vec : {1, full}) {
    if (q->channels % vec) continue;
    GnParams p = base_params(q);
    set_lanes(&p, vec);
    set_slabs(&p, kMostCtas, (backward ? 3 : 2) * q->pixels * q->channels * dtype_size(q->dtype));
    size_t n = gpart_bytes(p, p.S);
    if (backward) n += sizeof(float2) * kMostCtas * static_cast<size_t>(p.lanes) * vec;
    most = std::max(most, n);
  }
  return most;
}

int launch_group_norm_forward(const bevk_group_norm_problem *q, const void *x, const void *w,
                              const void *b, void *y, float *mean, float *rstd, void *ws,
                              size_t ws_bytes, cudaStream_t stream) {
  GnParams p = base_params(q);
  p.x = x;
  p.w = w;
  p.b = b;
  p.out = y;
  p.mean = mean;
  p.rstd = rstd;
  const int64_t size = dtype_size(q->dtype);
  const bool vectors = q->channels * size % 16 == 0 && vector_rows(x, q->input_strides, size) &&
                       vector_rows(y, q->output_strides, size);
  switch (q->dtype) {
    case BEVK_DTYPE_F16: return dispatch<__half>(p, false, vectors, ws, ws_bytes, stream);
    case BEVK_DTYPE_BF16: return dispatch<__nv_bfloat16>(p, false, vectors, ws, ws_bytes, stream);
    default: return dispatch<float>(p, false, vectors, ws, ws_bytes, stream);
  }
}

int launch_group_norm_backward(const bevk_group_norm_problem *q, const void *dy, const void *x,
                               const float *mean, const float *rstd, const void *w, const void *b,
                               void *dx, void *dw, void *db, void *ws, size_t ws_bytes,
                               cudaStream_t stream) {
  GnParams p = base_params(q);
  p.x = x;
  p.dy = dy;
  p.w = w;
  p.b = b;
  p.out = dx;
  p.dw = dw;
  p.db = db;
  p.mean = const_cast<float *>(mean);
  p.rstd = const_cast<float *>(rstd);
  const int64_t size = dtype_size(q->dtype);
  const bool vectors = q->channels * size % 16 == 0 && vector_rows(x, q->input_strides, size) &&
                       vector_rows(dy, q->grad_output_strides, size) &&
                       (dx == nullptr || vector_rows(dx, q->output_strides, size));
  switch (q->dtype) {
    case BEVK_DTYPE_F16: return dispatch<__half>(p, true, vectors, ws, ws_bytes, stream);
    case BEVK_DTYPE_BF16: return dispatch<__nv_bfloat16>(p, true, vectors, ws, ws_bytes, stream);
    default: return dispatch<float>(p, true, vectors, ws, ws_bytes, stream);
  }
}

}  // namespace bevk
