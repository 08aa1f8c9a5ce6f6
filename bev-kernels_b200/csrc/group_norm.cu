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
// launch and the reduction's latency when they are small.  One launch does both
// sweeps (cooperative, unless an image's CTAs make one cluster).  Every CTA owns
// a slab of pixels of one image (all channels where C allows): consecutive
// threads take consecutive 16-byte channel vectors, so a warp reads whole lines,
// and a thread keeps the same channels throughout (its weights stay in
// registers).  After the first sweep each CTA leaves one partial result per
// group, the CTAs meet, and each joins the partials of its own image in a fixed
// order before its second sweep.
//
// Every thread copies its own vectors to shared memory asynchronously -- all
// of them at once, without registers, and without synchronising with other
// threads -- and both sweeps read them there.  Images are taken in waves of
// up to twice what the SMs hold together (28 MB); the copies of the next wave
// follow the second sweep of this one into the slots that it has done with.
// The part of a slab that does not fit is read directly, twice.
//
// The variance is not a difference of large sums: a thread sums x - pivot and
// its square around the mean of its own first values, and the threads' (count,
// mean, M2) are joined by taking the mean of the means and then the squared
// deviations from it.  That holds when the mean is far from zero and when
// single values are far out.
//
// Device time, forward / backward (inputs in L2 where they fit; 16-bit unless
// said; bytes are the 2 and 3 passes): 1x64x32x32 fp32 ReLU 6.4 / 8.3 us; 6x512x29x50
// ReLU 9.8 (1.8 TB/s) / 14.8; 6x256x58x100 SiLU 14.1 / 26.3 us (2.5 / 2.0 TB/s);
// 1x256x200x200 fp32 SiLU 17.3 / 43 us (4.7 / 2.9); 12x256x116x200 SiLU 91 / 174 us
// (3.1 / 2.5).  The small ones are the latency of launch, load, reduction, meeting
// and store, about 1 to 1.5 us each.  Of a wave of the largest, 22 % (backward) and
// 23 % (forward) go to partial results, meeting and join, in which nothing moves:
// there is one CTA an SM, and all go through the steps together.  The second sweep,
// 57 % of a forward wave, writes, and fetches the next wave, at 4.9 TB/s together.
// Without an activation the large backward takes 136 us: SiLU's instructions, in
// both of its sweeps, are the rest.
//
// A wave has an image per CTA at most, so many small images are many waves: 1000 x
// 256 x 7 x 7 bf16 take 36 / 39 us (floor 8 / 12), 20000 x 256 single pixels, one of
// 16 rows of threads at work, 567 / 449 us (3 / 5).
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "bevk_internal.h"
#include "bevk_ptx.cuh"
#include "vec_io.cuh"

namespace cg = cooperative_groups;

namespace bevk {
namespace {

// Threads of a CTA.  More of them leave each too few registers: 1024 (forward)
// and 768 (backward) measured 1.2 to 1.5 times the time, with spills.  With 512 the
// 16-bit backward spills 12 bytes with SiLU, and 80 to 204 where vectors cross groups
// (6x264x58x100 bf16 SiLU of 24 groups 33.2 us, of 256 channels in 32 groups 25.8).
constexpr int kForwardThreads = 512;
constexpr int kBackwardThreads = 512;
constexpr int kBatch = 8;  // vectors of one asynchronous group, or loaded directly
constexpr int kPairs = 4;  // the backward's: x and dy
// Shared memory of a CTA; what the reductions leave of it holds vectors.
constexpr size_t kSmemBytes = 224 << 10;
// CTAs of a launch at most (one per SM): the workspace is sized for them.
constexpr int kMostCtas = 160;

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
  int nb;              // channel blocks
  int lanes, R;        // threads across a block's channels, rows of pixels
  int row_team, row_team_log;  // largest power of two <= R, at most team
  int team, team_log;  // threads that share a group (a power of two)
  int Gb;              // most groups that a channel block touches
  int wave;            // images per wave
  int cluster;         // 1: an image's CTAs are one thread-block cluster
  int S;               // slabs per image: `longer` of slab + 1 pixels, then of slab
  int slab, longer;
  int keep;            // vectors (backward: pairs) per thread held in shared memory
  int param_dtype, param_vectors;  // whether 16-byte loads fit weight and bias
  int slab_rows, slab_more;    // slab / R, slab % R
  int parts;                   // row classes that the channel sums are taken in first
  float inv_lanes, inv_k, inv_pitch;
  float eps;
};

// n / d for 0 <= n < 2^24 and inv = 1.f / d: a float quotient is off by one at
// most.  (The compiler's integer division is several times as long, and these
// stand in front of the first load.)
__device__ __forceinline__ int quotient(int n, int d, float inv) {
  int q = static_cast<int>(static_cast<float>(n) * inv);
  const int r = n - q * d;
  if (r < 0) --q;
  if (r >= d) ++q;
  return q;
}

// 1 / d of a count, and 1 / sqrt(v): the approximation and a Newton step, in
// place of the exact division and root, which stand on the critical path.
__device__ __forceinline__ float reciprocal(float d) {
  const float y = __fdividef(1.f, d);
  return fmaf(y, fmaf(-d, y, 1.f), y);
}
__device__ __forceinline__ float reciprocal_root(float v) {
  const float y = rsqrtf(v);
  const float z = fmaf(0.5f * y, fmaf(-v * y, y, 1.f), y);
  return v > 0.f && z == z ? z : y;  // 0 and infinity have their limits
}

// Sum over the w neighbouring lanes of a team (w a power of two); all get it.
__device__ __forceinline__ float team_sum(float v, int w) {
  for (int m = 1; m < w; m <<= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float exp2_approx(float t) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  return e;
}

// 1 / (1 + e^-z).  The special-function unit delivers a quarter of the other
// units' rate, and with two of its results a value (exponential, reciprocal)
// it would bound the 16-bit kernels.  So those take the reciprocal of
// d = 1 + e^-z = 2^E (1 + m) from a guess that is linear in m, which a
// subtraction from d's bits gives: y d = (1 + m)(2 - m - s) / 2 with the shift
// s = 5 - sqrt(24) that makes the error the same at m = 0 and in the middle
// (s / 2 = 5 %).  A third-order step, y (1 + h + h^2) with h = 1 - y d, and a
// Newton step leave (0.05^3)^2 = 1.7e-8, less than the two units of 2^-24 that the
// roundings add: the parameters' gradients are fp32 sums even where the tensors are
// not.  fp32 tensors get the hardware's reciprocal, and the rounding of -z log2(e)
// back to first order (at |z| = 10 that is five times the exponential's own error of
// 2^-22).
// z is at least kLowest, where d is 2^126.5, the most that the guess's bits stand
// for.  From d = 2^126 on 1 / d is subnormal, and both ways flush it to zero, so
// that z sigmoid(z) is zero however far below kLowest z was.
constexpr float kLowest = -87.68f;
template <typename T>
__device__ __forceinline__ vio::Two sigmoid(vio::Two z) {
  constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
  const vio::Two t2 = vio::mul2(z, vio::two(-kLog2e));
  const float2 t = vio::split(t2);
  if constexpr (sizeof(T) == 4) {
    const float2 f = vio::split(z);
    // (where t is infinite this is a NaN or too large, and counts nothing: e^-z is 0)
    const float lx = fminf(fmaf(f.x, -kLog2e, -t.x), 1.f), ly = fminf(fmaf(f.y, -kLog2e, -t.y), 1.f);
    float ex = exp2_approx(t.x), ey = exp2_approx(t.y);
    ex = fmaf(ex, lx * kLn2, ex);
    ey = fmaf(ey, ly * kLn2, ey);
    float sx, sy;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(sx) : "f"(1.f + ex));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(sy) : "f"(1.f + ey));
    return vio::two(sx, sy);
  } else {
    const float ex = exp2_approx(t.x), ey = exp2_approx(t.y);
    // -d, whose sign bit the guess's constant takes off again
    const vio::Two one = vio::two(1.f);
    const vio::Two minus = vio::fma2(vio::two(ex, ey), vio::two(-1.f), vio::two(-1.f));
    const float2 m = vio::split(minus);
    constexpr unsigned kGuess = 0x7ef311c3u + 0x80000000u;  // (254 - s) 2^23, and the sign
    vio::Two y = vio::two(__uint_as_float(kGuess - __float_as_uint(m.x)),
                          __uint_as_float(kGuess - __float_as_uint(m.y)));
    const vio::Two h = vio::fma2(minus, y, one);
    y = vio::fma2(y, vio::fma2(h, h, h), y);
    return vio::fma2_ftz(y, vio::fma2(minus, y, one), y);
  }
}
// z, or kLowest where z is below that; a NaN stays
__device__ __forceinline__ vio::Two from_lowest(vio::Two z) {
  const float2 f = vio::split(z);
  return vio::two(max_nan(f.x, kLowest), max_nan(f.y, kLowest));
}
template <typename T, int ACT>
__device__ __forceinline__ vio::Two activate(vio::Two z) {
  if constexpr (ACT == BEVK_ACT_RELU) {
    const float2 f = vio::split(z);
    return vio::two(f.x < 0.f ? 0.f : f.x, f.y < 0.f ? 0.f : f.y);  // NaN stays
  }
  if constexpr (ACT == BEVK_ACT_SILU) {
    z = from_lowest(z);
    return vio::mul2(z, sigmoid<T>(z));
  }
  return z;
}
// d act'(z); ReLU's slope is 0 at 0, SiLU's at infinity the formula's inf * 0 (its
// limit 1, by clamping z above too, cost 2 % of the backward)
template <typename T, int ACT>
__device__ __forceinline__ vio::Two through(vio::Two z, vio::Two d) {
  if constexpr (ACT == BEVK_ACT_RELU) {
    const float2 f = vio::split(z), g = vio::split(d);
    return vio::two(f.x > 0.f ? g.x : 0.f, f.y > 0.f ? g.y : 0.f);
  }
  if constexpr (ACT == BEVK_ACT_SILU) {
    z = from_lowest(z);
    const vio::Two s = sigmoid<T>(z);
    const vio::Two rest = vio::fma2(s, vio::two(-1.f), vio::two(1.f));
    return vio::mul2(d, vio::fma2(vio::mul2(z, s), rest, s));
  }
  return d;
}

// Where a thread stands: the same pixels of every wave's image, the same
// channels.
struct Place {
  int cb, s, image;       // channel block, slab, image within the wave
  int c0, c, bch;         // the block's first channel, the thread's, the block's count
  int r, lane;            // row of pixels, lane across the channels
  int p0, count;          // the slab
  int whole, more;        // rows < more hold whole + 1 of its pixels, the others whole
  int mine;               // pixels of this thread
  int g0, ng;             // groups that the block touches
  bool active;            // whether the thread has channels
};
__device__ __forceinline__ int slab_pixels(const GnParams &p, int s) {
  return p.slab + (s < p.longer ? 1 : 0);
}
template <int VEC>
__device__ __forceinline__ Place place(const GnParams &p) {
  Place t;
  int q = blockIdx.x;
  t.cb = 0;
  if (p.nb > 1) {
    t.cb = q % p.nb;
    q /= p.nb;
  }
  t.image = 0;
  if (p.wave > 1) {
    t.image = q / p.S;
    q -= t.image * p.S;
  }
  t.s = q;
  t.r = quotient(threadIdx.x, p.lanes, p.inv_lanes);
  t.lane = threadIdx.x - t.r * p.lanes;
  t.c0 = t.cb * p.lanes * VEC;
  t.c = t.c0 + t.lane * VEC;
  t.bch = min(p.C - t.c0, p.lanes * VEC);
  t.active = t.r < p.R && t.c < p.C;
  t.p0 = t.s * p.slab + min(t.s, p.longer);
  t.count = slab_pixels(p, t.s);
  t.whole = p.slab_rows;
  t.more = p.slab_more + (t.count - p.slab);
  if (t.more == p.R) {
    ++t.whole;
    t.more = 0;
  }
  t.mine = t.active ? t.whole + (t.r < t.more ? 1 : 0) : 0;
  t.g0 = quotient(t.c0, p.K, p.inv_k);
  t.ng = quotient(t.c0 + t.bch - 1, p.K, p.inv_k) + 1 - t.g0;
  return t;
}

// The partials of group g of image n: entry e of [0, count) lies in channel
// block cb0 + e / S, slab e % S.  (A group spans several blocks only where its
// channels do not fit one.)
struct Partials {
  const float2 *base;
  int g, cb0, bw, count;
};
__device__ __forceinline__ Partials partials_of(const GnParams &p, int n, int g, int bw) {
  if (p.nb == 1) return {p.gpart + (static_cast<int64_t>(n) * p.Gb + g) * p.S, g, 0, bw, p.S};
  const int cb0 = g * p.K / bw, cb1 = ((g + 1) * p.K - 1) / bw;
  return {p.gpart + static_cast<int64_t>(n) * p.nb * p.Gb * p.S, g, cb0, bw,
          (cb1 - cb0 + 1) * p.S};
}
// Entry e, and the number of values behind it.
__device__ __forceinline__ float2 partial(const GnParams &p, const Partials &q, int e,
                                          float *values) {
  if (p.nb == 1) {
    *values = static_cast<float>(slab_pixels(p, e)) * p.K;
    return __ldcg(q.base + e);
  }
  const int b = e / p.S, cb = q.cb0 + b, s = e - b * p.S;
  const int c0 = cb * q.bw;
  *values = static_cast<float>(slab_pixels(p, s)) *
            (min((q.g + 1) * p.K, c0 + q.bw) - max(q.g * p.K, c0));
  return __ldcg(q.base + (static_cast<int64_t>(cb) * p.Gb + (q.g - c0 / p.K)) * p.S + s);
}
__device__ __forceinline__ float2 *partial_slot(const GnParams &p, const Place &t, int n, int gl) {
  return p.gpart + ((static_cast<int64_t>(n) * p.nb + t.cb) * p.Gb + gl) * p.S + t.s;
}

// Mean and rstd of the block's groups from the slabs' (mean, M2): first the
// mean of the means, then the squared deviations from it.  The threads of a
// team take the partials in turn and keep the first few in registers, so the
// loads are in flight together.
template <int kThreads>
__device__ void combine_moments(const GnParams &p, const Place &t, int n, int bw, float *s_mean,
                                float *s_rstd, bool write) {
  constexpr int kKeep = 10;
  const int w = p.team, j = threadIdx.x & (w - 1);
  const float inv = reciprocal(static_cast<float>(p.HW) * p.K);
  for (int base = 0; base < t.ng; base += kThreads >> p.team_log) {
    const int gl = base + (threadIdx.x >> p.team_log);
    const bool on = gl < t.ng;
    const Partials q = partials_of(p, n, on ? t.g0 + gl : t.g0, bw);
    float2 v[kKeep];
    float c[kKeep];
#pragma unroll
    for (int k = 0; k < kKeep; ++k) {
      v[k] = make_float2(0.f, 0.f);
      c[k] = 0.f;
      if (on && j + k * w < q.count) v[k] = partial(p, q, j + k * w, &c[k]);
    }
    float sum = 0.f, m2 = 0.f, u;
#pragma unroll
    for (int k = 0; k < kKeep; ++k) sum += c[k] * v[k].x;
    for (int e = j + kKeep * w; on && e < q.count; e += w) sum += partial(p, q, e, &u).x * u;
    const float mean = team_sum(sum, w) * inv;
#pragma unroll
    for (int k = 0; k < kKeep; ++k) m2 += v[k].y + c[k] * (v[k].x - mean) * (v[k].x - mean);
    for (int e = j + kKeep * w; on && e < q.count; e += w) {
      const float2 f = partial(p, q, e, &u);
      m2 += f.y + u * (f.x - mean) * (f.x - mean);
    }
    m2 = team_sum(m2, w);
    if (on && j == 0) {
      const float rstd = reciprocal_root(fmaf(m2, inv, p.eps));
      s_mean[gl] = mean;
      s_rstd[gl] = rstd;
      if (write) {
        p.mean[static_cast<int64_t>(n) * p.G + t.g0 + gl] = mean;
        p.rstd[static_cast<int64_t>(n) * p.G + t.g0 + gl] = rstd;
      }
    }
  }
}

// The sums' counterpart for the backward.
template <int kThreads>
__device__ void combine_sums(const GnParams &p, const Place &t, int n, int bw, float inv_m,
                             float2 *s_sum) {
  constexpr int kKeep = 10;
  const int w = p.team, j = threadIdx.x & (w - 1);
  for (int base = 0; base < t.ng; base += kThreads >> p.team_log) {
    const int gl = base + (threadIdx.x >> p.team_log);
    const bool on = gl < t.ng;
    const Partials q = partials_of(p, n, on ? t.g0 + gl : t.g0, bw);
    float2 v[kKeep];
    float u;
#pragma unroll
    for (int k = 0; k < kKeep; ++k) {
      v[k] = make_float2(0.f, 0.f);
      if (on && j + k * w < q.count) v[k] = partial(p, q, j + k * w, &u);
    }
    float a = 0.f, b = 0.f;
#pragma unroll
    for (int k = 0; k < kKeep; ++k) {
      a += v[k].x;
      b += v[k].y;
    }
    for (int e = j + kKeep * w; on && e < q.count; e += w) {
      const float2 f = partial(p, q, e, &u);
      a += f.x;
      b += f.y;
    }
    a = team_sum(a, w);
    b = team_sum(b, w);
    if (on && j == 0) s_sum[gl] = make_float2(a * inv_m, b * inv_m);
  }
}

// Whether a vector goes to shared memory by asynchronous 16-byte copies (else
// through registers).
template <typename T, int VEC>
constexpr bool kAsync = sizeof(T) * VEC == 16;

template <typename T, int VEC>
__device__ __forceinline__ void fetch(char *slot, const T *src) {
  if constexpr (kAsync<T, VEC>) vio::copy_async<16>(slot, src);
  else vio::store_pack<T, VEC>(slot, vio::load_pack<T, VEC>(src));
}

template <typename T, int VEC, bool WHOLE, int ACT>
__global__ void __launch_bounds__(kForwardThreads, 1)
    gn_forward_kernel(const __grid_constant__ GnParams p) {
  constexpr int kThreads = kForwardThreads;
  // statistics columns of a thread: one where its vector lies in one group,
  // else one per channel
  constexpr int NC = WHOLE ? 1 : VEC;
  constexpr int CH = VEC / NC;
  constexpr int kBytes = sizeof(T) * VEC;
  using Vec = vio::Pack<T, VEC>;
  extern __shared__ float4 s_dyn[];
  const int tid = threadIdx.x;
  char *s_mine = reinterpret_cast<char *>(s_dyn) + tid * kBytes;  // [keep][kThreads] vectors
  constexpr int kSlot = kThreads * kBytes;
  float2 *s_red = reinterpret_cast<float2 *>(reinterpret_cast<char *>(s_dyn) + p.keep * kSlot);
  float *s_mean = reinterpret_cast<float *>(s_red + (kThreads + p.lanes) * NC);
  float *s_rstd = s_mean + p.Gb;  // [Gb] each
  cg::grid_group grid = cg::this_grid();

  ptx::grid_launch_dependents();
  ptx::grid_wait_prerequisites();
  const Place t = place<VEC>(p);
  const int held = min(t.mine, p.keep);
  const int groups = (p.keep + kBatch - 1) / kBatch;  // asynchronous ones, of every thread
  const int64_t hop = static_cast<int64_t>(p.R) * p.xs[1];
  const int64_t out_hop = static_cast<int64_t>(p.R) * p.os[1];
  int n = t.image;
  const T *src = static_cast<const T *>(p.x) + n * p.xs[0] +
                 static_cast<int64_t>(t.p0 + t.r) * p.xs[1] + t.c;
  T *dst = static_cast<T *>(p.out) + n * p.os[0] + static_cast<int64_t>(t.p0 + t.r) * p.os[1] + t.c;
  for (int g = 0; g < groups; ++g) {
    for (int i = g * kBatch; i < min(held, (g + 1) * kBatch) && n < p.N; ++i)
      fetch<T, VEC>(s_mine + i * kSlot, src + i * hop);
    vio::copy_commit();
  }

  for (int n0 = 0; n0 < p.N; n0 += p.wave) {
    if (n < p.N) {
      // sums of x - pivot and its square, the two values of a pair apart; the
      // pivot is the mean of the first group
      constexpr int P = vio::kPairsOf<VEC>;
      float pivot[NC];
      vio::Two minus[NC == 1 ? 1 : P], sum2[NC == 1 ? 1 : P], sq2[NC == 1 ? 1 : P];
#pragma unroll
      for (int k = 0; k < NC; ++k) pivot[k] = 0.f;
#pragma unroll
      for (int k = 0; k < (NC == 1 ? 1 : P); ++k) sum2[k] = sq2[k] = vio::two(0.f);
      const auto aim = [&](const Vec &q) {
        float f[VEC];
        vio::unpack(q, f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) pivot[e / CH] += f[e];
      };
      const auto aimed = [&](float count) {
        const float inv = reciprocal(count * CH);
#pragma unroll
        for (int k = 0; k < NC; ++k) pivot[k] *= inv;
#pragma unroll
        for (int k = 0; k < (NC == 1 ? 1 : P); ++k)
          minus[k] = vio::two(-pivot[NC == 1 ? 0 : 2 * k],
                              VEC == 1 ? 0.f : -pivot[NC == 1 ? 0 : 2 * k + 1]);
      };
      const auto add = [&](const Vec &q) {
        vio::Two f[P];
        vio::unpack2<T, VEC>(q, f);
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const int k = NC == 1 ? 0 : i;
          const vio::Two d = vio::add2(f[i], minus[k]);
          sum2[k] = vio::add2(sum2[k], d);
          sq2[k] = vio::fma2(d, d, sq2[k]);
        }
      };
      const auto slot = [&](int i) { return vio::load_pack<T, VEC>(s_mine + i * kSlot); };
      for (int g = 0; g < groups; ++g) {
        vio::copy_wait(groups - 1 - g);
        const int i1 = min(held, (g + 1) * kBatch);
        if (g == 0) {
#pragma unroll 4
          for (int i = 0; i < i1; ++i) aim(slot(i));
          aimed(static_cast<float>(max(i1, 1)));
        }
#pragma unroll 4
        for (int i = g * kBatch; i < i1; ++i) add(slot(i));
      }
      for (int i0 = held; i0 < t.mine; i0 += kBatch) {  // what is not held
        Vec v[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
          if (i0 + i < t.mine) v[i] = vio::load_pack<T, VEC>(src + (i0 + i) * hop);
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
          if (i0 + i < t.mine) add(v[i]);
      }
      // s_red: [statistics column][lane][row], rows padded to an odd number: the
      // threads of a warp write a row and read a column without bank conflicts
      const int pitch = p.R | 1;
      if (t.active) {
        const float inv = reciprocal(static_cast<float>(max(t.mine, 1) * CH));
#pragma unroll
        for (int k = 0; k < NC; ++k) {
          const float2 s2 = vio::split(sum2[NC == 1 ? 0 : k / 2]);
          const float2 q2 = vio::split(sq2[NC == 1 ? 0 : k / 2]);
          const float sum = VEC == 1 ? s2.x : NC == 1 ? s2.x + s2.y : k % 2 ? s2.y : s2.x;
          const float sq = VEC == 1 ? q2.x : NC == 1 ? q2.x + q2.y : k % 2 ? q2.y : q2.x;
          // squares that overflow leave an infinite variance, not a NaN
          const float m2 = isinf(sq) ? sq : sq - sum * (sum * inv);
          s_red[(k * p.lanes + t.lane) * pitch + t.r] =
              make_float2(pivot[k] + sum * inv, m2 < 0.f ? 0.f : m2);
        }
      }
      __syncthreads();
      // one team per group joins the rows and columns of the group: the mean
      // of the means, then the squared deviations from it
      const int w = p.team, j = tid & (w - 1);
      const int wr = p.row_team, jr = j & (wr - 1), jc = j >> p.row_team_log;
      const int wc = w >> p.row_team_log;
      const int rows = t.whole ? p.R : t.more;
      for (int base = 0; base < t.ng; base += kThreads >> p.team_log) {
        const int gl = base + (tid >> p.team_log);
        int k0 = 0, k1 = 0;
        if (gl < t.ng) {
          k0 = max((t.g0 + gl) * p.K - t.c0, 0) / CH;
          k1 = min((t.g0 + gl + 1) * p.K - t.c0, t.bch) / CH;
        }
        const auto at = [&](int row, int k) {  // column k: lane k / NC, entry k % NC
          return s_red[((k % NC) * p.lanes + k / NC) * pitch + row];
        };
        float s = 0.f, m2 = 0.f;
        for (int row = jr; row < rows; row += wr) {
          const float c = static_cast<float>((t.whole + (row < t.more ? 1 : 0)) * CH);
          for (int k = k0 + jc; k < k1; k += wc) s += c * at(row, k).x;
        }
        const float mean =
            team_sum(s, w) * reciprocal(static_cast<float>(t.count) * max((k1 - k0) * CH, 1));
        for (int row = jr; row < rows; row += wr) {
          const float c = static_cast<float>((t.whole + (row < t.more ? 1 : 0)) * CH);
          for (int k = k0 + jc; k < k1; k += wc) {
            const float2 v = at(row, k);
            m2 += v.y + c * (v.x - mean) * (v.x - mean);
          }
        }
        m2 = team_sum(m2, w);
        if (gl < t.ng && j == 0) __stcg(partial_slot(p, t, n, gl), make_float2(mean, m2));
      }
    }
    const auto pw = vio::load_params<VEC>(t.active ? p.w : nullptr, t.c, p.param_dtype,
                                           p.param_vectors != 0);
    const auto pb = vio::load_params<VEC>(t.active ? p.b : nullptr, t.c, p.param_dtype,
                                           p.param_vectors != 0);
    if (p.S == 1 && p.nb == 1) __syncthreads();
    else if (p.cluster) ptx::cluster_sync();
    else grid.sync();
    const bool next = n + p.wave < p.N;
    if (n < p.N) {
      combine_moments<kThreads>(p, t, n, p.lanes * VEC, s_mean, s_rstd,
                                p.mean != nullptr && t.s == 0);
      __syncthreads();
      float a[VEC], b[VEC];  // z = a x + b
      vio::params_to_float(pw, p.w, p.param_dtype, 1.f, a);
      vio::params_to_float(pb, p.b, p.param_dtype, 0.f, b);
      if (t.mine > 0) {
#pragma unroll
        for (int k = 0; k < NC; ++k) {
          const int gl = quotient(t.c + k * CH, p.K, p.inv_k) - t.g0;
          const float mean = s_mean[gl], rstd = s_rstd[gl];
#pragma unroll
          for (int e = k * CH; e < (k + 1) * CH; ++e) {
            a[e] *= rstd;
            b[e] = fmaf(-mean, a[e], b[e]);
          }
        }
      }
      constexpr int P = vio::kPairsOf<VEC>;
      vio::Two a2[P], b2[P];
#pragma unroll
      for (int i = 0; i < P; ++i) {
        a2[i] = VEC == 1 ? vio::two(a[0], 0.f) : vio::two(a[2 * i], a[VEC == 1 ? 0 : 2 * i + 1]);
        b2[i] = VEC == 1 ? vio::two(b[0], 0.f) : vio::two(b[2 * i], b[VEC == 1 ? 0 : 2 * i + 1]);
      }
      const auto write = [&](const Vec &q, int i) {
        vio::Two v[P];
        vio::unpack2<T, VEC>(q, v);
#pragma unroll
        for (int e = 0; e < P; ++e) v[e] = activate<T, ACT>(vio::fma2(v[e], a2[e], b2[e]));
        vio::store2<T, VEC>(dst + i * out_hop, v);
      };
      const T *src1 = src + p.wave * p.xs[0];
      for (int g = 0; g < groups; ++g) {
#pragma unroll 4
        for (int i = g * kBatch; i < min(held, (g + 1) * kBatch); ++i) {
          write(vio::load_pack<T, VEC>(s_mine + i * kSlot), i);
          if (next) fetch<T, VEC>(s_mine + i * kSlot, src1 + i * hop);
        }
        vio::copy_commit();
      }
#pragma unroll 4
      for (int i = held; i < t.mine; ++i) write(vio::load_pack<T, VEC>(src + i * hop), i);
      src = src1;
      dst += p.wave * p.os[0];
    }
    n += p.wave;
  }
}

template <typename T, int VEC, bool WHOLE, int ACT>
__global__ void __launch_bounds__(kBackwardThreads, 1)
    gn_backward_kernel(const __grid_constant__ GnParams p) {
  constexpr int kThreads = kBackwardThreads;
  constexpr int NC = WHOLE ? 1 : VEC;  // groups that a thread's vector may touch
  constexpr int CH = VEC / NC;
  constexpr int kBytes = sizeof(T) * VEC;
  using Vec = vio::Pack<T, VEC>;
  extern __shared__ float4 s_dyn[];
  const int tid = threadIdx.x;
  char *s_mine = reinterpret_cast<char *>(s_dyn) + tid * kBytes;  // [keep][x, dy][kThreads]
  constexpr int kSlot = kThreads * kBytes;
  float2 *s_red = reinterpret_cast<float2 *>(reinterpret_cast<char *>(s_dyn) + 2 * p.keep * kSlot);
  float2 *s_tot = s_red + kThreads * VEC;  // s_red: [R][lanes * VEC]; s_tot: over all waves
  float2 *s_sum = s_tot + p.lanes * VEC;   // [Gb] s1 / m, s2 / m
  float *s_w = reinterpret_cast<float *>(s_sum + p.Gb);  // [lanes * VEC]
  // per-channel arrays hold element e of lane l at e * lanes + l
  const auto entry = [&](int channel) { return channel % VEC * p.lanes + channel / VEC; };
  cg::grid_group grid = cg::this_grid();

  const Place t = place<VEC>(p);
  const int held = min(t.mine, p.keep);
  const int groups = (p.keep + kPairs - 1) / kPairs;
  const int64_t xhop = static_cast<int64_t>(p.R) * p.xs[1];
  const int64_t ghop = static_cast<int64_t>(p.R) * p.gs[1];
  const int64_t out_hop = static_cast<int64_t>(p.R) * p.os[1];
  const int64_t row0 = t.p0 + t.r;
  int n = t.image;
  const T *px = static_cast<const T *>(p.x) + n * p.xs[0] + row0 * p.xs[1] + t.c;
  const T *pg = static_cast<const T *>(p.dy) + n * p.gs[0] + row0 * p.gs[1] + t.c;
  T *dst = static_cast<T *>(p.out) + n * p.os[0] + row0 * p.os[1] + t.c;
  for (int g = 0; g < groups; ++g) {
    for (int i = g * kPairs; i < min(held, (g + 1) * kPairs) && n < p.N; ++i) {
      fetch<T, VEC>(s_mine + 2 * i * kSlot, px + i * xhop);
      fetch<T, VEC>(s_mine + (2 * i + 1) * kSlot, pg + i * ghop);
    }
    vio::copy_commit();
  }
  float w[VEC], b[VEC];
  {
    const auto pw = vio::load_params<VEC>(t.active ? p.w : nullptr, t.c, p.param_dtype,
                                           p.param_vectors != 0);
    const auto pb = vio::load_params<VEC>(t.active ? p.b : nullptr, t.c, p.param_dtype,
                                           p.param_vectors != 0);
    vio::params_to_float(pw, p.w, p.param_dtype, 1.f, w);
    vio::params_to_float(pb, p.b, p.param_dtype, 0.f, b);
  }
  if (t.active && t.r == 0) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) s_w[e * p.lanes + t.lane] = w[e];
  }
  constexpr int P = vio::kPairsOf<VEC>;
  vio::Two w2[P], b2[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    w2[i] = VEC == 1 ? vio::two(w[0], 0.f) : vio::two(w[2 * i], w[VEC == 1 ? 0 : 2 * i + 1]);
    b2[i] = VEC == 1 ? vio::two(b[0], 0.f) : vio::two(b[2 * i], b[VEC == 1 ? 0 : 2 * i + 1]);
  }
  // the pair's groups
  const auto pair_of = [](const float (&v)[NC], int i) {
    return NC == 1 ? vio::two(v[0]) : vio::two(v[NC == 1 ? 0 : 2 * i], v[NC == 1 ? 0 : 2 * i + 1]);
  };
  int group[NC];
#pragma unroll
  for (int k = 0; k < NC; ++k) group[k] = quotient(t.c + k * CH, p.K, p.inv_k);
  const int pitch = p.lanes * VEC;  // s_red's rows (entries of absent lanes are never used)
  for (int k = tid; k < pitch; k += kThreads) s_tot[k] = make_float2(0.f, 0.f);
  const float inv_m = 1.f / (static_cast<float>(p.K) * static_cast<float>(p.HW));
  const bool params = p.dw != nullptr || p.db != nullptr;

  for (int n0 = 0; n0 < p.N; n0 += p.wave) {
    float rstd[NC], shift[NC];  // xhat = rstd x + shift
    if (n < p.N) {
      vio::Two A[P], B[P];
#pragma unroll
      for (int e = 0; e < P; ++e) A[e] = B[e] = vio::two(0.f);
#pragma unroll
      for (int k = 0; k < NC; ++k) {
        const int64_t g = static_cast<int64_t>(n) * p.G + group[k];
        rstd[k] = t.active ? p.rstd[g] : 0.f;
        shift[k] = t.active ? -p.mean[g] * rstd[k] : 0.f;
      }
      const auto add = [&](const Vec &qx, const Vec &qg) {
        vio::Two f[P], d[P];
        vio::unpack2<T, VEC>(qx, f);
        vio::unpack2<T, VEC>(qg, d);
#pragma unroll
        for (int e = 0; e < P; ++e) {
          const vio::Two xhat = vio::fma2(f[e], pair_of(rstd, e), pair_of(shift, e));
          const vio::Two dz = through<T, ACT>(vio::fma2(xhat, w2[e], b2[e]), d[e]);
          A[e] = vio::add2(A[e], dz);
          B[e] = vio::fma2(dz, xhat, B[e]);
        }
      };
      for (int i0 = held; i0 < t.mine; i0 += kPairs) {
        Vec qx[kPairs], qg[kPairs];
#pragma unroll
        for (int i = 0; i < kPairs; ++i)
          if (i0 + i < t.mine) {
            qx[i] = vio::load_pack<T, VEC>(px + (i0 + i) * xhop);
            qg[i] = vio::load_pack<T, VEC>(pg + (i0 + i) * ghop);
          }
#pragma unroll
        for (int i = 0; i < kPairs; ++i)
          if (i0 + i < t.mine) add(qx[i], qg[i]);
      }
      for (int g = 0; g < groups; ++g) {
        vio::copy_wait(groups - 1 - g);
#pragma unroll 2
        for (int i = g * kPairs; i < min(held, (g + 1) * kPairs); ++i)
          add(vio::load_pack<T, VEC>(s_mine + 2 * i * kSlot),
              vio::load_pack<T, VEC>(s_mine + (2 * i + 1) * kSlot));
      }
      if (t.active) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float2 a = vio::split(A[e / 2]), c = vio::split(B[e / 2]);
          s_red[t.r * pitch + e * p.lanes + t.lane] =
              e % 2 ? make_float2(a.y, c.y) : make_float2(a.x, c.x);
        }
      }
      __syncthreads();
      // channel sums over the rows, in two steps where threads are left over;
      // then row 0 of s_red holds w * sum
      if (p.parts > 1) {
        const int part = quotient(tid, pitch, p.inv_pitch), k = tid - part * pitch;
        if (part < p.parts) {
          float2 s = s_red[part * pitch + k];
#pragma unroll 4
          for (int row = part + p.parts; row < p.R; row += p.parts) {
            const float2 v = s_red[row * pitch + k];
            s.x += v.x;
            s.y += v.y;
          }
          s_red[part * pitch + k] = s;
        }
        __syncthreads();
      }
      for (int k = tid; k < pitch; k += kThreads) {
        float2 s = s_red[k];
#pragma unroll 4
        for (int row = 1; row < (p.parts > 1 ? p.parts : p.R); ++row) {
          const float2 v = s_red[row * pitch + k];
          s.x += v.x;
          s.y += v.y;
        }
        s_tot[k].x += s.x;
        s_tot[k].y += s.y;
        const float wk = s_w[k];
        s_red[k] = make_float2(s.x * wk, s.y * wk);
      }
      __syncthreads();
      const int j = tid & (p.team - 1);
      for (int base = 0; base < t.ng; base += kThreads >> p.team_log) {
        const int gl = base + (tid >> p.team_log);
        float s1 = 0.f, s2 = 0.f;
        if (gl < t.ng) {
          const int k0 = max((t.g0 + gl) * p.K - t.c0, 0);
          const int k1 = min((t.g0 + gl + 1) * p.K - t.c0, t.bch);
          for (int k = k0 + j; k < k1; k += p.team) {
            const float2 v = s_red[entry(k)];
            s1 += v.x;
            s2 += v.y;
          }
        }
        s1 = team_sum(s1, p.team);
        s2 = team_sum(s2, p.team);
        if (gl < t.ng && j == 0) __stcg(partial_slot(p, t, n, gl), make_float2(s1, s2));
      }
    }
    const bool last = n0 + p.wave >= p.N;
    if (last && params)
      for (int k = tid; k < pitch; k += kThreads)
        __stcg(p.cpart + static_cast<int64_t>(blockIdx.x) * p.lanes * VEC + k, s_tot[k]);
    if (p.S > 1 || p.nb > 1 || (last && params)) grid.sync();
    else __syncthreads();
    const bool next = n + p.wave < p.N;
    if (n < p.N) {
      const T *px1 = px + p.wave * p.xs[0], *pg1 = pg + p.wave * p.gs[0];
      if (p.out != nullptr) {
        combine_sums<kThreads>(p, t, n, p.lanes * VEC, inv_m, s_sum);
        __syncthreads();
        float r1[NC], r2[NC];  // dx = rstd w dz + r2 xhat + r1
#pragma unroll
        for (int k = 0; k < NC; ++k) {
          const float2 s = t.active ? s_sum[group[k] - t.g0] : make_float2(0.f, 0.f);
          r1[k] = -rstd[k] * s.x;
          r2[k] = -rstd[k] * s.y;
        }
        const auto write = [&](const Vec &qx, const Vec &qg, int i) {
          vio::Two f[P], d[P];
          vio::unpack2<T, VEC>(qx, f);
          vio::unpack2<T, VEC>(qg, d);
#pragma unroll
          for (int e = 0; e < P; ++e) {
            const vio::Two xhat = vio::fma2(f[e], pair_of(rstd, e), pair_of(shift, e));
            const vio::Two dz = through<T, ACT>(vio::fma2(xhat, w2[e], b2[e]), d[e]);
            f[e] = vio::fma2(vio::mul2(pair_of(rstd, e), w2[e]), dz,
                             vio::fma2(xhat, pair_of(r2, e), pair_of(r1, e)));
          }
          vio::store2<T, VEC>(dst + i * out_hop, f);
        };
        for (int g = 0; g < groups; ++g) {
#pragma unroll 2
          for (int i = g * kPairs; i < min(held, (g + 1) * kPairs); ++i) {
            char *slot = s_mine + 2 * i * kSlot;
            write(vio::load_pack<T, VEC>(slot), vio::load_pack<T, VEC>(slot + kSlot), i);
            if (next) {
              fetch<T, VEC>(slot, px1 + i * xhop);
              fetch<T, VEC>(slot + kSlot, pg1 + i * ghop);
            }
          }
          vio::copy_commit();
        }
#pragma unroll 2
        for (int i = held; i < t.mine; ++i)
          write(vio::load_pack<T, VEC>(px + i * xhop), vio::load_pack<T, VEC>(pg + i * ghop), i);
      } else if (next) {
        for (int g = 0; g < groups; ++g) {
          for (int i = g * kPairs; i < min(held, (g + 1) * kPairs); ++i) {
            fetch<T, VEC>(s_mine + 2 * i * kSlot, px1 + i * xhop);
            fetch<T, VEC>(s_mine + (2 * i + 1) * kSlot, pg1 + i * ghop);
          }
          vio::copy_commit();
        }
      }
      px = px1;
      pg = pg1;
      dst += p.wave * p.os[0];
    }
    n += p.wave;
  }
  // grad_weight and grad_bias: 32 channels at a time, the CTAs' sums in order
  if (!params) return;
  __syncthreads();
  const int wl = tid & 31, wid = tid >> 5;
  const int bw = p.lanes * VEC;
  for (int base = blockIdx.x * 32; base < p.C; base += gridDim.x * 32) {
    const int ch = base + wl;
    float2 s = make_float2(0.f, 0.f);
    if (ch < p.C) {
      const int blk = ch / bw, k = entry(ch - blk * bw);
#pragma unroll 10
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
#pragma unroll 5
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
// error), remembered per kernel and device.
template <auto kernel>
int resident_ctas(int threads) {
  static thread_local int seen_device = -1, seen_ctas = 0;
  const int dev = current_device();
  if (dev < 0) return 0;
  if (seen_device == dev) return seen_ctas;
  int per_sm = 0;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           static_cast<int>(kSmemBytes)) != cudaSuccess ||
      cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, kSmemBytes) !=
          cudaSuccess)
    return 0;
  seen_ctas = std::min(kMostCtas, per_sm * device_info(dev).sm_count);
  seen_device = dev;
  return seen_ctas;
}

constexpr int threads_of(bool back) { return back ? kBackwardThreads : kForwardThreads; }

// Channels across the threads of a CTA: everything that follows from the
// shape, the types and the vector width alone.
void set_lanes(GnParams *p, int vec, int kThreads) {
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
  p->team = 32;
  p->team_log = 5;
  while (p->team > 1 && p->team * p->Gb > kThreads) {
    p->team >>= 1;
    --p->team_log;
  }
  p->row_team = 1;
  p->row_team_log = 0;
  while (2 * p->row_team <= std::min(p->R, p->team)) {
    p->row_team *= 2;
    ++p->row_team_log;
  }
  p->inv_lanes = 1.f / p->lanes;
  p->inv_k = 1.f / p->K;
  p->parts = std::min(p->R, std::max(1, kThreads / (p->lanes * vec)));
  p->inv_pitch = 1.f / (p->lanes * vec);
}

// Pixels per slab at least two for every thread: the most slabs of an image.
int most_slabs(const GnParams &p) {
  return static_cast<int>(std::max<int64_t>(1, p.HW / (static_cast<int64_t>(p.R) * 2)));
}

// Waves and slabs for `ctas` resident CTAs, each with room for `room` vectors
// of every thread; returns the grid, one CTA per (image of a wave, slab,
// channel block).  A wave is as many images as make twice what the CTAs hold, at
// least one; the waves are then made equal.  What is not held is read twice, the
// second time from L2; against waves that are held whole, fewer meetings of the
// grid gain more, and three times as much gains and loses.  SiLU, forward /
// backward in us with once, twice, three times what is held:
//   12x256x116x200 bf16    91 / 197    91 / 174   108 / 176
//   12x256x116x200 fp32   164 / 274   167 / 273   201 / 273
//   7x256x116x200 bf16     63 / 118    60 / 118    66 / 127
//   13x256x58x100 bf16     29 / 69     22 / 56     22 / 50
//   6x256x58x100 fp32      20 / 40     16 / 36     16 / 33
//   4x256x200x200 fp32     93 / 175    93 / 175   114 / 175
// (one image is one wave: 1x256x400x400 bf16 65 / 109, 1x256x300x300 fp32 69 / 106).
int set_slabs(GnParams *p, int ctas, int room) {
  const int64_t image = (p->HW + p->R - 1) / p->R;  // vectors of a thread for a whole image
  const int64_t most = std::max<int64_t>(
      1, std::min<int64_t>(ctas / p->nb, 2 * ctas * static_cast<int64_t>(room) / (image * p->nb)));
  const int64_t waves = (p->N + most - 1) / most;
  p->wave = static_cast<int>((p->N + waves - 1) / waves);
  const int64_t cut = most_slabs(*p);
  p->S = static_cast<int>(
      std::max<int64_t>(1, std::min<int64_t>(ctas / (static_cast<int64_t>(p->wave) * p->nb), cut)));
  p->slab = p->HW / p->S;
  p->longer = p->HW - p->slab * p->S;
  p->slab_rows = p->slab / p->R;
  p->slab_more = p->slab - p->slab_rows * p->R;
  const int slab = p->slab + (p->longer ? 1 : 0);
  p->keep = std::min(room, (slab + p->R - 1) / p->R);
  return p->wave * p->nb * p->S;
}

// Bytes of shared memory besides the vectors, and the room that is left.
size_t reduce_bytes(const GnParams &p, int vec, bool back) {
  const int kThreads = threads_of(back);
  if (back)
    return sizeof(float2) * (static_cast<size_t>(kThreads) * vec + p.lanes * vec + p.Gb) +
           sizeof(float) * p.lanes * vec;
  return sizeof(float2) * ((kThreads + p.lanes) * (p.K % vec == 0 ? 1 : vec) + p.Gb);
}
int room_for(size_t reduce, size_t bytes_per_slot, int threads) {
  return static_cast<int>((kSmemBytes - reduce) / (bytes_per_slot * threads));
}

size_t gpart_bytes(const GnParams &p) {
  return sizeof(float2) * static_cast<size_t>(p.N) * p.nb * p.Gb * p.S;
}

// Where every image's CTAs can be one cluster, with all clusters resident, they
// meet at the cluster's barrier instead of the grid's, and the launch is an
// ordinary one.  That has fewer CTAs than the grid, so it pays while each has
// little to do: measured against the grid (device time), 64x32x32 f32 6.4 and
// 7.4 us, 30x128x28x28 bf16 10.6 and 11.6, 6x512x29x50 f16 (12 vectors a thread)
// 9.8 and 9.9, but 1x256x58x100 bf16 (24 vectors) 15.7 and 9.1.
// Sets the slabs and returns true where it is used.  (The forward's alone: the backward
// ends in channel sums over all CTAs, behind a meeting of the grid.)
constexpr int kMostHeldByCluster = 12;
template <auto kernel>
bool set_clusters(GnParams *p, int room) {
  if (p->nb > 1) return false;
  static thread_local int seen_device = -1, fits[17];
  const int dev = current_device();
  if (seen_device != dev) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) {
      (void)cudaGetLastError();
      return false;
    }
    for (int c : {1, 2, 4, 8, 16}) {
      cudaLaunchConfig_t cfg = {};
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = c;
      attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
      cfg.gridDim = dim3(c);
      cfg.blockDim = dim3(kForwardThreads);
      cfg.dynamicSmemBytes = kSmemBytes;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&fits[c], kernel, &cfg) != cudaSuccess) {
        (void)cudaGetLastError();
        fits[c] = 0;
      }
    }
    seen_device = dev;
  }
  const int cut = most_slabs(*p);
  for (int c : {16, 8, 4, 2, 1}) {
    if (fits[c] < p->N) continue;
    const int S = std::min(c, cut);
    const int slab = (p->HW + S - 1) / S, keep = (slab + p->R - 1) / p->R;
    if (keep > std::min(room, kMostHeldByCluster)) return false;
    p->S = S;
    p->wave = p->N;
    p->slab = p->HW / S;
    p->longer = p->HW - p->slab * S;
    p->slab_rows = p->slab / p->R;
    p->slab_more = p->slab - p->slab_rows * p->R;
    p->keep = keep;
    p->cluster = 1;
    return true;
  }
  return false;
}

template <auto kernel>
int launch(GnParams p, int vec, size_t size, bool back, void *ws, size_t ws_bytes,
           cudaStream_t stream) {
  const int threads = threads_of(back);
  const int ctas = resident_ctas<kernel>(threads);
  if (ctas <= 0) return fail(BEVK_ERR_CUDA, "group_norm_act: occupancy query failed");
  if (ctas < p.nb)
    return fail(BEVK_ERR_UNSUPPORTED, "group_norm_act: %d channels are too many", p.C);
  p.param_vectors = aligned(p.w, 16) && aligned(p.b, 16);
  const size_t reduce = reduce_bytes(p, vec, back);
  const size_t slot = (back ? 2 : 1) * vec * size;
  const int room = room_for(reduce, slot, threads);
  int grid = set_slabs(&p, ctas, room);
  const bool clusters = !back && set_clusters<kernel>(&p, room);
  if (clusters) grid = p.N * p.S;
  const size_t cpart = back ? static_cast<size_t>(grid) * p.lanes * vec : 0;
  const size_t need = cpart * sizeof(float2) + gpart_bytes(p);
  if (ws_bytes < need)
    return fail(BEVK_ERR_WORKSPACE, "group_norm_act: workspace of %zu bytes, needs %zu", ws_bytes,
                need);
  p.cpart = static_cast<float2 *>(ws);
  p.gpart = p.cpart + cpart;
  if (clusters) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = p.S;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = reduce + p.keep * slot * threads;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = programmatic_launch_enabled() ? 2 : 1;
    return launched(cudaLaunchKernelEx(&cfg, kernel, p), "gn_forward_kernel");
  }
  void *args[] = {&p};
  return launched(cudaLaunchCooperativeKernel(reinterpret_cast<void *>(kernel), dim3(grid),
                                              dim3(threads), args, reduce + p.keep * slot * threads,
                                              stream),
                  back ? "gn_backward_kernel" : "gn_forward_kernel");
}

template <typename T, int ACT>
int dispatch(GnParams &p, bool back, bool vectors, void *ws, size_t ws_bytes,
             cudaStream_t stream) {
  constexpr int V = vio::Full<T>::value;
  const int vec = vectors ? V : 1;
  set_lanes(&p, vec, threads_of(back));
  const auto run = [&](auto kernel) {
    return launch<decltype(kernel)::value>(p, vec, sizeof(T), back, ws, ws_bytes, stream);
  };
#define BEVK_GN_RUN(...) run(std::integral_constant<void (*)(GnParams), __VA_ARGS__>())
  if (!vectors)
    return back ? BEVK_GN_RUN(gn_backward_kernel<T, 1, true, ACT>)
                : BEVK_GN_RUN(gn_forward_kernel<T, 1, true, ACT>);
  if (p.K % V == 0)
    return back ? BEVK_GN_RUN(gn_backward_kernel<T, V, true, ACT>)
                : BEVK_GN_RUN(gn_forward_kernel<T, V, true, ACT>);
  return back ? BEVK_GN_RUN(gn_backward_kernel<T, V, false, ACT>)
              : BEVK_GN_RUN(gn_forward_kernel<T, V, false, ACT>);
#undef BEVK_GN_RUN
}
template <typename T>
int dispatch(GnParams &p, int act, bool back, bool vectors, void *ws, size_t ws_bytes,
             cudaStream_t stream) {
  switch (act) {
    case BEVK_ACT_RELU: return dispatch<T, BEVK_ACT_RELU>(p, back, vectors, ws, ws_bytes, stream);
    case BEVK_ACT_SILU: return dispatch<T, BEVK_ACT_SILU>(p, back, vectors, ws, ws_bytes, stream);
    default: return dispatch<T, BEVK_ACT_NONE>(p, back, vectors, ws, ws_bytes, stream);
  }
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
  p.eps = q->eps;
  return p;
}

int dispatch(const bevk_group_norm_problem *q, GnParams &p, bool back, bool vectors, void *ws,
             size_t ws_bytes, cudaStream_t stream) {
  switch (q->dtype) {
    case BEVK_DTYPE_F16:
      return dispatch<__half>(p, q->act, back, vectors, ws, ws_bytes, stream);
    case BEVK_DTYPE_BF16:
      return dispatch<__nv_bfloat16>(p, q->act, back, vectors, ws, ws_bytes, stream);
    default: return dispatch<float>(p, q->act, back, vectors, ws, ws_bytes, stream);
  }
}

}  // namespace

size_t group_norm_workspace_bytes(const bevk_group_norm_problem *q, bool backward) {
  // whichever vector width the call takes, and however many CTAs it gets: an
  // image has at most kMostCtas / nb slabs, and a launch kMostCtas CTAs
  size_t most = 0;
  const int size = static_cast<int>(dtype_size(q->dtype));
  for (int vec : {1, 16 / size}) {
    if (q->channels % vec) continue;
    GnParams p = base_params(q);
    set_lanes(&p, vec, threads_of(backward));
    const int64_t cut = most_slabs(p);
    p.S = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(kMostCtas / p.nb, cut)));
    size_t n = gpart_bytes(p);
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
  return dispatch(q, p, false, vectors, ws, ws_bytes, stream);
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
  return dispatch(q, p, true, vectors, ws, ws_bytes, stream);
}

}  // namespace bevk
