// embedding.cu -- embedding lookup with scaling and its gradient.
//
//   forward   y_i = s W[id_i]
//   backward  dW[v] (+)= s sum_{i : id_i = v} dy_i
//
// The lookup moves num_ids * dim elements twice and computes nothing to speak
// of: 16-byte vectors, several rows in flight per thread.
//
// The gradient is a sum over tokens per table row, with rows that no id names
// (most of a vocabulary) and rows that thousands of ids name.  Atomics into
// the table would make the sums' order, and so their last bits, change from
// run to run, and would serialise on the frequent rows.  Here the tokens are
// ordered by id (a stable radix sort), and the ordered list is cut into tiles
// of 32 tokens.  Every warp takes one tile of one slice of the columns -- the
// same work whatever the ids are -- and walks it in order with fp32 sums in
// registers.  A run of equal ids that lies inside its tile is finished there;
// the pieces of a run that crosses tiles go to scratch and a last kernel adds
// them in order.  The sort runs on one thread-block cluster (its passes meet
// at the cluster's hardware barrier, keys and positions stay in L2) while the
// other SMs write the zeros of a dense gradient, which are most of its bytes.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "bevk_internal.h"
#include "bevk_ptx.cuh"
#include "vec_io.cuh"

namespace bevk {
namespace {

// ------------------------------------------------------------------ forward
constexpr int kLookThreads = 256;
constexpr int kLookRows = 4;  // rows a thread has in flight

struct LookParams {
  const void *table, *ids;
  void *out;
  int64_t ld, n, rows;
  int dim, tx;  // tx threads side by side on a row (a power of two)
  float scale;
};

template <typename T, typename Id, int VEC>
__global__ void __launch_bounds__(kLookThreads) embedding_forward_kernel(const LookParams p) {
  ptx::grid_launch_dependents();
  ptx::grid_wait_prerequisites();
  const int tx = threadIdx.x & (p.tx - 1), ty = threadIdx.x / p.tx;
  const int step = kLookThreads / p.tx;  // rows side by side in a CTA
  const T *table = static_cast<const T *>(p.table);
  const Id *ids = static_cast<const Id *>(p.ids);
  T *out = static_cast<T *>(p.out);
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * step * kLookRows; base < p.n;
       base += static_cast<int64_t>(gridDim.x) * step * kLookRows) {
    int64_t id[kLookRows];
#pragma unroll
    for (int k = 0; k < kLookRows; ++k) {
      const int64_t r = base + k * step + ty;
      id[k] = r < p.n ? static_cast<int64_t>(ids[r]) : -1;
      if (id[k] >= p.rows) id[k] = -1;
    }
    for (int c = tx * VEC; c < p.dim; c += p.tx * VEC) {
      float v[kLookRows][VEC];
#pragma unroll
      for (int k = 0; k < kLookRows; ++k) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[k][e] = 0.f;
        if (id[k] >= 0) vio::unpack(vio::load_pack<T, VEC>(table + id[k] * p.ld + c), v[k]);
      }
#pragma unroll
      for (int k = 0; k < kLookRows; ++k) {
        const int64_t r = base + k * step + ty;
        if (r >= p.n) continue;
        if (id[k] >= 0) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) v[k][e] *= p.scale;
        }
        vio::store<T, VEC>(out + r * p.dim + c, v[k]);
      }
    }
  }
}

// ----------------------------------------------------------------- sorting
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kDigits = 256;
constexpr int kMostCluster = 16;
constexpr int kTile = 32;  // tokens of one tile of the ordered list

struct Owner {  // a run of equal ids that goes on past the tile it begins in
  unsigned tile, slot;
};

struct SortParams {
  const void *ids;
  unsigned *key[2], *pos[2];
  unsigned *hist;     // [cluster size][kDigits]
  unsigned *owners;   // how many
  Owner *owner;
  int64_t rows, padding;
  int n, passes, cluster;
  // zeros of a dense gradient: rows of row_bytes at pitch bytes
  char *zero;
  int64_t zero_rows, row_bytes, pitch;
};

// An id as a sort key; what gets no gradient sorts behind all rows.
template <typename Id>
__device__ __forceinline__ unsigned key_of(Id id, const SortParams &p) {
  const int64_t v = static_cast<int64_t>(id);
  return v >= 0 && v < p.rows && v != p.padding ? static_cast<unsigned>(v)
                                                : static_cast<unsigned>(p.rows);
}

__device__ void write_zeros(const SortParams &p, int part, int parts) {
  const int64_t t = static_cast<int64_t>(part) * kSortThreads + threadIdx.x;
  const int64_t threads = static_cast<int64_t>(parts) * kSortThreads;
  const bool flat = p.row_bytes == p.pitch;
  const int64_t rows = flat ? 1 : p.zero_rows;
  const int64_t bytes = flat ? p.zero_rows * p.row_bytes : p.row_bytes;
  if (reinterpret_cast<uintptr_t>(p.zero) % 16 == 0 && bytes % 16 == 0 &&
      (flat || p.pitch % 16 == 0)) {
    const int64_t vecs = bytes / 16;
    for (int64_t i = t; i < rows * vecs; i += threads) {
      const int64_t r = flat ? 0 : i / vecs;
      *reinterpret_cast<uint4 *>(p.zero + r * p.pitch + (i - r * vecs) * 16) = make_uint4(0, 0, 0, 0);
    }
  } else {  // elements of two bytes at least
    const int64_t halves = bytes / 2;
    for (int64_t i = t; i < rows * halves; i += threads) {
      const int64_t r = flat ? 0 : i / halves;
      *reinterpret_cast<uint16_t *>(p.zero + r * p.pitch + (i - r * halves) * 2) = 0;
    }
  }
}

template <typename Id>
__global__ void __launch_bounds__(kSortThreads) embedding_sort_kernel(const SortParams p) {
  __shared__ unsigned s_cnt[kSortWarps][kDigits];
  __shared__ unsigned s_scan[kDigits];
  ptx::grid_launch_dependents();
  ptx::grid_wait_prerequisites();
  if (static_cast<int>(blockIdx.x) >= p.cluster) {
    write_zeros(p, blockIdx.x - p.cluster, gridDim.x - p.cluster);
    return;
  }
  const int rank = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (rank == 0 && tid == 0) *p.owners = 0;
  // this CTA's tokens, and this warp's part of them, in order
  const int b0 = static_cast<int>(static_cast<int64_t>(p.n) * rank / p.cluster);
  const int b1 = static_cast<int>(static_cast<int64_t>(p.n) * (rank + 1) / p.cluster);
  const int chunk = ((b1 - b0 + kSortThreads - 1) / kSortThreads) * 32;
  const int w0 = min(b1, b0 + warp * chunk), w1 = min(b1, w0 + chunk);
  const Id *ids = static_cast<const Id *>(p.ids);

  for (int pass = 0; pass < p.passes; ++pass) {
    const unsigned *kin = p.key[(pass + 1) & 1], *pin = p.pos[(pass + 1) & 1];
    unsigned *kout = p.key[pass & 1], *pout = p.pos[pass & 1];
    const int shift = 8 * pass;
    for (int i = tid; i < kSortWarps * kDigits; i += kSortThreads) (&s_cnt[0][0])[i] = 0;
    __syncthreads();
    // digits of the warp's tokens
    for (int i = w0 + lane; i - lane < w1; i += 32) {
      const unsigned active = __ballot_sync(0xffffffffu, i < w1);
      if (i < w1) {
        const unsigned k = pass ? __ldcg(kin + i) : key_of(ids[i], p);
        const unsigned d = (k >> shift) & (kDigits - 1);
        const unsigned same = __match_any_sync(active, d);
        if (lane == __ffs(same) - 1) s_cnt[warp][d] += __popc(same);
      }
      __syncwarp();
    }
    __syncthreads();
    // digit totals of the CTA, over the cluster
    if (tid < kDigits) {
      unsigned sum = 0;
      for (int w = 0; w < kSortWarps; ++w) sum += s_cnt[w][tid];
      __stcg(p.hist + rank * kDigits + tid, sum);
    }
    ptx::cluster_sync();
    unsigned before = 0, total = 0;
    if (tid < kDigits) {
      for (int r = 0; r < p.cluster; ++r) {
        const unsigned h = __ldcg(p.hist + r * kDigits + tid);
        if (r < rank) before += h;
        total += h;
      }
      s_scan[tid] = total;
    }
    __syncthreads();
    for (int m = 1; m < kDigits; m <<= 1) {  // inclusive scan over the digits
      unsigned v = 0;
      if (tid < kDigits && tid >= m) v = s_scan[tid - m];
      __syncthreads();
      if (tid < kDigits) s_scan[tid] += v;
      __syncthreads();
    }
    if (tid < kDigits) {
      unsigned at = s_scan[tid] - total + before;
      for (int w = 0; w < kSortWarps; ++w) {
        const unsigned c = s_cnt[w][tid];
        s_cnt[w][tid] = at;
        at += c;
      }
    }
    __syncthreads();
    for (int i = w0 + lane; i - lane < w1; i += 32) {
      const unsigned active = __ballot_sync(0xffffffffu, i < w1);
      if (i < w1) {
        const unsigned k = pass ? __ldcg(kin + i) : key_of(ids[i], p);
        const unsigned d = (k >> shift) & (kDigits - 1);
        const unsigned same = __match_any_sync(active, d);
        const unsigned at = s_cnt[warp][d] + __popc(same & ((1u << lane) - 1));
        __syncwarp(active);
        if (lane == __ffs(same) - 1) s_cnt[warp][d] += __popc(same);
        kout[at] = k;
        pout[at] = pass ? __ldcg(pin + i) : static_cast<unsigned>(i);
      }
      __syncwarp();
    }
    ptx::cluster_sync();
  }
  // runs that go on past the tile they begin in
  const unsigned *key = p.key[(p.passes + 1) & 1];
  const int tiles = (p.n + kTile - 1) / kTile;
  for (int t = rank * kSortThreads + tid; t < tiles; t += p.cluster * kSortThreads) {
    const int64_t last = static_cast<int64_t>(t) * kTile + kTile - 1;
    if (last + 1 >= p.n) continue;
    const unsigned k = __ldcg(key + last);
    if (k >= static_cast<unsigned>(p.rows) || __ldcg(key + last + 1) != k) continue;
    if (t > 0 && __ldcg(key + static_cast<int64_t>(t) * kTile - 1) == k) continue;
    const unsigned slot = __ldcg(key + static_cast<int64_t>(t) * kTile) == k ? 0u : 1u;
    p.owner[atomicAdd(p.owners, 1u)] = {static_cast<unsigned>(t), slot};  // any order will do
  }
}

// -------------------------------------------------------------------- sums
struct SumParams {
  const void *dy;
  void *out;
  const unsigned *key, *pos;
  const unsigned *owners;
  const Owner *owner;
  float *partial;    // [tile][2][pdim]: a run's piece at the tile's start, or further in
  int64_t dy_ld, out_ld;
  int n, rows, dim, pdim, slices;
  float scale;
  int accumulate;
};

// The finished sums of VEC columns, 16 bytes of the output at a time.
template <typename O, int VEC>
__device__ __forceinline__ void finish(const SumParams &p, unsigned row, int c,
                                       const float (&v)[VEC]) {
  constexpr int P = VEC < vio::Full<O>::value ? VEC : vio::Full<O>::value;
  O *dst = static_cast<O *>(p.out) + static_cast<int64_t>(row) * p.out_ld + c;
  float old[VEC];
  if (p.accumulate) {
#pragma unroll
    for (int k = 0; k < VEC; k += P) {
      float f[P];
      vio::unpack(vio::load_pack<O, P>(dst + k), f);
#pragma unroll
      for (int e = 0; e < P; ++e) old[k + e] = f[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) old[e] = 0.f;
  }
#pragma unroll
  for (int k = 0; k < VEC; k += P) {
    float f[P];
#pragma unroll
    for (int e = 0; e < P; ++e) f[e] = fmaf(v[k + e], p.scale, old[k + e]);
    vio::store<O, P>(dst + k, f);
  }
}

constexpr int kSumThreads = 256;
constexpr int kAhead = 8;  // rows loaded before they are used

// One warp per (tile, slice of 32 * VEC columns).
template <typename T, typename O, int VEC>
__global__ void __launch_bounds__(kSumThreads) embedding_sum_kernel(const SumParams p) {
  ptx::grid_launch_dependents();
  ptx::grid_wait_prerequisites();
  const int lane = threadIdx.x & 31;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * (kSumThreads / 32) + (threadIdx.x >> 5);
  const int64_t tile = item / p.slices;
  const int c = (static_cast<int>(item - tile * p.slices) * 32 + lane) * VEC;
  const int64_t first = tile * kTile;
  if (first >= p.n) return;
  const bool have = first + lane < p.n;
  const unsigned none = static_cast<unsigned>(p.rows);
  const unsigned key = have ? p.key[first + lane] : none;
  const unsigned pos = have ? p.pos[first + lane] : 0u;
  const unsigned before = first > 0 ? p.key[first - 1] : none;
  const unsigned after = first + kTile < p.n ? p.key[first + kTile] : none;
  const int count = __popc(__ballot_sync(0xffffffffu, key != none));  // rows come first
  const unsigned next = __shfl_down_sync(0xffffffffu, key, 1);
  // bit j: token j is the last of its run within the tile
  const unsigned ends = __ballot_sync(0xffffffffu, lane == 31 || key != next);
  const T *dy = static_cast<const T *>(p.dy) + c;
  const bool col = c < p.dim;
  float acc[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
  int begin = 0;
  for (int j0 = 0; j0 < count; j0 += kAhead) {
    vio::Pack<T, VEC> q[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const unsigned at = __shfl_sync(0xffffffffu, pos, (j0 + j) & 31);
      if (col && j0 + j < count)
        q[j] = vio::load_pack<T, VEC>(dy + static_cast<int64_t>(at) * p.dy_ld);
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int t = j0 + j;
      if (t >= count) break;
      if (col) {
        float v[VEC];
        vio::unpack(q[j], v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] += v[e];
      }
      if ((ends >> t) & 1u) {
        const unsigned row = __shfl_sync(0xffffffffu, key, t);
        const bool open = (begin == 0 && before == row) || (t == kTile - 1 && after == row);
        if (col) {
          if (open) {
            float *dst = p.partial + (tile * 2 + (begin ? 1 : 0)) * p.pdim + c;
#pragma unroll
            for (int e = 0; e < VEC; ++e) __stcg(dst + e, acc[e]);
          } else {
            finish<O, VEC>(p, row, c, acc);
          }
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
        begin = t + 1;
      }
    }
  }
}

// Runs that cross tiles: a CTA adds the pieces of one run for 128 columns,
// each warp a stretch of them in order, then the warps' sums in order.
template <typename O>
__global__ void __launch_bounds__(kSumThreads) embedding_join_kernel(const SumParams p) {
  constexpr int kWarps = kSumThreads / 32;
  __shared__ float4 s_sum[kWarps][32];
  ptx::grid_launch_dependents();
  ptx::grid_wait_prerequisites();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int slices = (p.pdim + 127) / 128;
  const int64_t items = static_cast<int64_t>(*p.owners) * slices;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const Owner o = p.owner[item / slices];
    const int c = static_cast<int>(item % slices) * 128 + lane * 4;
    const int64_t first = static_cast<int64_t>(o.tile) * kTile;
    const unsigned row = p.key[first + kTile - 1];
    // tiles after o.tile whose first token is still of this run
    int more = 0;
    for (;;) {
      const int64_t t = (o.tile + 1 + static_cast<int64_t>(more) + lane) * kTile;
      const unsigned on = __ballot_sync(0xffffffffu, t < p.n && p.key[t] == row);
      const int run = on == 0xffffffffu ? 32 : __ffs(~on) - 1;
      more += run;
      if (run < 32) break;
    }
    const int pieces = more + 1;
    const int per = (pieces + kWarps - 1) / kWarps;
    const int a = min(pieces, warp * per), b = min(pieces, a + per);
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (c < p.pdim) {
      const float *src = p.partial + c;
#pragma unroll 8
      for (int k = a; k < b; ++k) {
        const int64_t at = (static_cast<int64_t>(o.tile) + k) * 2 + (k == 0 ? o.slot : 0u);
        const float4 v = __ldcg(reinterpret_cast<const float4 *>(src + at * p.pdim));
        s.x += v.x;
        s.y += v.y;
        s.z += v.z;
        s.w += v.w;
      }
    }
    s_sum[warp][lane] = s;
    __syncthreads();
    if (warp == 0) {
      for (int w = 1; w < kWarps; ++w) {
        const float4 v = s_sum[w][lane];
        s.x += v.x;
        s.y += v.y;
        s.z += v.z;
        s.w += v.w;
      }
      const float f[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (c + e < p.dim) {
          float one[1] = {f[e]};
          finish<O, 1>(p, row, c + e, one);
        }
      }
    }
    __syncthreads();
  }
}

// -------------------------------------------------------------------- host
template <typename T, int VEC>
int look(const LookParams &p0, bool wide_ids, cudaStream_t stream) {
  LookParams p = p0;
  p.tx = 1;
  while (p.tx < kLookThreads && p.tx * VEC < p.dim) p.tx <<= 1;
  const int64_t rows = static_cast<int64_t>(kLookThreads / p.tx) * kLookRows;
  const int64_t want = (p.n + rows - 1) / rows;
  const int dev = current_device();
  if (dev < 0) return fail(BEVK_ERR_CUDA, "embedding_forward: no device");
  const int grid = static_cast<int>(std::min<int64_t>(want, int64_t(64) * device_info(dev).sm_count));
  return launched(wide_ids ? launch_dependent(embedding_forward_kernel<T, int64_t, VEC>, dim3(grid),
                                              dim3(kLookThreads), 0, stream, p)
                           : launch_dependent(embedding_forward_kernel<T, int32_t, VEC>, dim3(grid),
                                              dim3(kLookThreads), 0, stream, p),
                  "embedding_forward_kernel");
}

template <typename T>
int look_any(const LookParams &p, bool wide_ids, cudaStream_t stream) {
  constexpr int V = vio::Full<T>::value;
  const bool vectors = p.dim % V == 0 && p.ld % V == 0 && aligned(p.table, 16) && aligned(p.out, 16);
  return vectors ? look<T, V>(p, wide_ids, stream) : look<T, 1>(p, wide_ids, stream);
}

struct Layout {  // of the backward's workspace
  size_t key[2], pos[2], hist, owners, owner, partial, bytes;
  int64_t tiles;
  int pdim;
};
Layout layout_of(const bevk_embedding_backward_args *a) {
  Layout l;
  size_t at = 0;
  const auto take = [&at](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  const size_t n = static_cast<size_t>(a->num_ids);
  l.tiles = (a->num_ids + kTile - 1) / kTile;
  l.pdim = (a->dim + 3) / 4 * 4;
  for (int i = 0; i < 2; ++i) {
    l.key[i] = take(n * 4);
    l.pos[i] = take(n * 4);
  }
  l.hist = take(sizeof(unsigned) * kMostCluster * kDigits);
  l.owners = take(sizeof(unsigned));
  l.owner = take(sizeof(Owner) * static_cast<size_t>(l.tiles));
  l.partial = take(sizeof(float) * 2 * static_cast<size_t>(l.tiles) * l.pdim);
  l.bytes = at;
  return l;
}

// CTAs of the sorting cluster: 4096 tokens each up to the hardware's most
// (16 where a cluster of that size fits on the device, else 8).
int cluster_size(int64_t n) {
  int c = 1;
  while (c < kMostCluster && n > int64_t(4096) * c) c <<= 1;
  return c;
}

template <typename Id>
int sort_ids(const SortParams &p0, bool dense, cudaStream_t stream) {
  SortParams p = p0;
  const int dev = current_device();
  if (dev < 0) return fail(BEVK_ERR_CUDA, "embedding_backward: no device");
  auto kernel = embedding_sort_kernel<Id>;
  p.cluster = cluster_size(p.n);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.blockDim = dim3(kSortThreads);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = programmatic_launch_enabled() ? 2 : 1;
  cfg.gridDim = dim3(p.cluster);
  if (p.cluster > 8) {
    static thread_local int seen_device = -1, fits = 0;
    if (seen_device != dev) {
      const unsigned attrs = cfg.numAttrs;
      cfg.numAttrs = 1;
      if (cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) !=
              cudaSuccess ||
          cudaOccupancyMaxActiveClusters(&fits, kernel, &cfg) != cudaSuccess) {
        (void)cudaGetLastError();
        fits = 0;
      }
      cfg.numAttrs = attrs;
      seen_device = dev;
    }
    if (fits < 1) attr[0].val.clusterDim.x = p.cluster = 8;
  }
  int grid = p.cluster;
  if (dense) {  // about an SM's worth of CTAs for every other SM, in whole clusters
    const int64_t bytes = p.zero_rows * p.row_bytes;
    const int64_t want = std::max<int64_t>(1, bytes / (64 * kSortThreads));
    const int64_t room = std::max(1, device_info(dev).sm_count - p.cluster);
    const int extra = static_cast<int>(std::min(want, room));
    grid += (extra + p.cluster - 1) / p.cluster * p.cluster;
  }
  cfg.gridDim = dim3(grid);
  return launched(cudaLaunchKernelEx(&cfg, kernel, p), "embedding_sort_kernel");
}

template <typename T, typename O, int VEC>
int sum(const SumParams &p0, int64_t tiles, cudaStream_t stream) {
  SumParams p = p0;
  p.slices = (p.dim + 32 * VEC - 1) / (32 * VEC);
  const int64_t warps = tiles * p.slices, per = kSumThreads / 32;
  const int64_t grid = (warps + per - 1) / per;
  if (grid >= (int64_t(1) << 31))
    return fail(BEVK_ERR_INDEX_OVERFLOW, "embedding_backward: too many tokens and columns");
  const int st = launched(launch_dependent(embedding_sum_kernel<T, O, VEC>,
                                           dim3(static_cast<unsigned>(grid)), dim3(kSumThreads), 0,
                                           stream, p),
                          "embedding_sum_kernel");
  if (st != BEVK_OK) return st;
  if (tiles < 2) return BEVK_OK;  // no run crosses tiles
  const int64_t items = (tiles - 1) * ((p.pdim + 127) / 128);
  const int64_t most = int64_t(4) * device_info(current_device()).sm_count;
  return launched(launch_dependent(embedding_join_kernel<O>,
                                   dim3(static_cast<unsigned>(std::min(items, most))),
                                   dim3(kSumThreads), 0, stream, p),
                  "embedding_join_kernel");
}

template <typename T, typename O>
int sum_any(const SumParams &p, int64_t tiles, cudaStream_t stream) {
  constexpr int V = vio::Full<T>::value;
  const bool vectors = p.dim % V == 0 && p.dy_ld % V == 0 &&
                       p.out_ld * sizeof(O) % 16 == 0 &&
                       aligned(p.dy, 16) && aligned(p.out, 16);
  return vectors ? sum<T, O, V>(p, tiles, stream) : sum<T, O, 1>(p, tiles, stream);
}

}  // namespace

int launch_embedding_forward(const void *table, int64_t ld, const void *ids, bool wide_ids,
                             int64_t n, int64_t rows, int dim, float scale, void *out, int dtype,
                             cudaStream_t stream) {
  const LookParams p = {table, ids, out, ld, n, rows, dim, 0, scale};
  switch (dtype) {
    case BEVK_DTYPE_F16: return look_any<__half>(p, wide_ids, stream);
    case BEVK_DTYPE_BF16: return look_any<__nv_bfloat16>(p, wide_ids, stream);
    default: return look_any<float>(p, wide_ids, stream);
  }
}

size_t embedding_backward_workspace_bytes(const bevk_embedding_backward_args *a) {
  return layout_of(a).bytes;
}

int launch_embedding_backward(const bevk_embedding_backward_args *a, const void *dy,
                              const void *ids, void *grad_table, void *ws, cudaStream_t stream) {
  const Layout l = layout_of(a);
  char *base = static_cast<char *>(ws);
  SortParams s = {};
  s.ids = ids;
  for (int i = 0; i < 2; ++i) {
    s.key[i] = reinterpret_cast<unsigned *>(base + l.key[i]);
    s.pos[i] = reinterpret_cast<unsigned *>(base + l.pos[i]);
  }
  s.hist = reinterpret_cast<unsigned *>(base + l.hist);
  s.owners = reinterpret_cast<unsigned *>(base + l.owners);
  s.owner = reinterpret_cast<Owner *>(base + l.owner);
  s.rows = a->num_rows;
  s.padding = a->padding_idx;
  s.n = static_cast<int>(a->num_ids);
  s.passes = 1;
  while (s.passes < 4 && (a->num_rows >> (8 * s.passes)) != 0) ++s.passes;
  const int64_t size = dtype_size(a->grad_table_dtype);
  s.zero = static_cast<char *>(grad_table);
  s.zero_rows = a->num_rows;
  s.row_bytes = a->dim * size;
  s.pitch = a->grad_table_ld * size;
  const int st = a->ids_are_64bit ? sort_ids<int64_t>(s, !a->accumulate, stream)
                                  : sort_ids<int32_t>(s, !a->accumulate, stream);
  if (st != BEVK_OK) return st;
  SumParams p = {};
  p.dy = dy;
  p.out = grad_table;
  p.key = s.key[(s.passes + 1) & 1];
  p.pos = s.pos[(s.passes + 1) & 1];
  p.owners = s.owners;
  p.owner = s.owner;
  p.partial = reinterpret_cast<float *>(base + l.partial);
  p.dy_ld = a->grad_output_ld;
  p.out_ld = a->grad_table_ld;
  p.n = s.n;
  p.rows = static_cast<int>(a->num_rows);
  p.dim = a->dim;
  p.pdim = l.pdim;
  p.scale = a->scale;
  p.accumulate = a->accumulate;
  const bool wide = a->grad_table_dtype == BEVK_DTYPE_F32;
  switch (a->grad_output_dtype) {
    case BEVK_DTYPE_F16:
      return wide ? sum_any<__half, float>(p, l.tiles, stream)
                  : sum_any<__half, __half>(p, l.tiles, stream);
    case BEVK_DTYPE_BF16:
      return wide ? sum_any<__nv_bfloat16, float>(p, l.tiles, stream)
                  : sum_any<__nv_bfloat16, __nv_bfloat16>(p, l.tiles, stream);
    default: return sum_any<float, float>(p, l.tiles, stream);
  }
}

}  // namespace bevk
