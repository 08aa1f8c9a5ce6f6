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
// them in order.  The sort runs on one thread-block cluster: its passes meet
// at the cluster's hardware barrier and exchange their digit totals through
// distributed shared memory, the list stays in L2.  The zeros of a dense
// gradient, most of its bytes, are written by another kernel at the same time.
//
// Bound by memory at many tokens (writes alone reach 3.7 to 4 TB/s on this part,
// reads 5 at these sizes), by the chain of launches and the sort at few.
// Device time: 65536 rows of 4 KB looked up in 61 us (333 MB, 5.4 TB/s); their
// gradient added to 10000 fp32 rows in 130 us (430 MB; the sort 20 us of it);
// 16384 tokens into a dense 50021 x 1024 bf16 table in 41 us (136 MB); 40000
// tokens of 200 rows of 512 bytes in 17 us, of which the sort is 9; 30 tokens in
// 12 us, the launches of zeros, sort and sums.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

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
    // single elements are taken four at a time, so that as many loads are on
    // their way
    constexpr int W = VEC == 1 ? 4 : 1;
    for (int c0 = tx * VEC; c0 < p.dim; c0 += p.tx * VEC * W) {
      float v[kLookRows][W][VEC];
#pragma unroll
      for (int k = 0; k < kLookRows; ++k) {
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const int c = c0 + w * p.tx;
#pragma unroll
          for (int e = 0; e < VEC; ++e) v[k][w][e] = 0.f;
          if (id[k] >= 0 && c < p.dim)
            vio::unpack(vio::load_pack<T, VEC>(table + id[k] * p.ld + c), v[k][w]);
        }
      }
#pragma unroll
      for (int k = 0; k < kLookRows; ++k) {
        const int64_t r = base + k * step + ty;
        if (r >= p.n) continue;
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const int c = c0 + w * p.tx;
          if (id[k] >= 0) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[k][w][e] *= p.scale;
          }
          if (c < p.dim) vio::store<T, VEC>(out + r * p.dim + c, v[k][w]);
        }
      }
    }
  }
}

// ----------------------------------------------------------------- sorting
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kDigits = 256;
constexpr int kMostCluster = 16;
constexpr int kTile = 32;   // tokens of one tile of the ordered list
constexpr int kShort = 8;   // pieces of a run that one warp joins

using Entry = unsigned long long;  // sort key << 32 | position
__host__ __device__ constexpr Entry entry_of(unsigned key, unsigned pos) {
  return static_cast<Entry>(key) << 32 | pos;
}
__device__ __forceinline__ unsigned key_in(Entry e) { return static_cast<unsigned>(e >> 32); }

struct ZeroParams {  // zeros of a dense gradient: rows of row_bytes at pitch bytes
  char *out;
  int64_t rows, row_bytes, pitch;
};

struct SortParams {
  const void *ids;
  Entry *list0, *list1;  // written by the even and the odd passes
  unsigned *count;       // [2], zeroed for the sums
  int64_t rows, padding;
  int n, passes, cluster;
  int behind_zeros;   // launched while embedding_zero_kernel runs
  ZeroParams zeros;   // of a table that is small enough to leave them to the sort (rows > 0)
};

// An id as a sort key; what gets no gradient sorts behind all rows.
template <typename Id>
__device__ __forceinline__ unsigned key_of(Id id, const SortParams &p) {
  const int64_t v = static_cast<int64_t>(id);
  return v >= 0 && v < p.rows && v != p.padding ? static_cast<unsigned>(v)
                                                : static_cast<unsigned>(p.rows);
}

// Writes thread `t` of `threads`' share of the zeros: 16 bytes at a time in one
// stretch of memory (its ends by halves: elements have two bytes at least) or in
// rows of whole 16-byte parts, else halves.
__device__ __forceinline__ void write_zeros(const ZeroParams &p, int64_t t, int64_t threads) {
  const uint4 zero = make_uint4(0, 0, 0, 0);
  if (p.row_bytes == p.pitch || p.rows == 1) {
    const int64_t bytes = p.rows * p.row_bytes;
    const int64_t head = min(bytes, static_cast<int64_t>(-reinterpret_cast<uintptr_t>(p.out) & 15));
    const int64_t vecs = (bytes - head) / 16, tail = head + vecs * 16;
    for (int64_t i = t; i < vecs; i += threads)
      *reinterpret_cast<uint4 *>(p.out + head + i * 16) = zero;
    if (2 * t < head) *reinterpret_cast<uint16_t *>(p.out + 2 * t) = 0;
    if (2 * t < bytes - tail) *reinterpret_cast<uint16_t *>(p.out + tail + 2 * t) = 0;
  } else if (reinterpret_cast<uintptr_t>(p.out) % 16 == 0 && p.row_bytes % 16 == 0 &&
             p.pitch % 16 == 0) {
    const int64_t vecs = p.row_bytes / 16;
    for (int64_t i = t; i < p.rows * vecs; i += threads) {
      const int64_t r = i / vecs;
      *reinterpret_cast<uint4 *>(p.out + r * p.pitch + (i - r * vecs) * 16) = zero;
    }
  } else {
    const int64_t halves = p.row_bytes / 2;
    for (int64_t i = t; i < p.rows * halves; i += threads) {
      const int64_t r = i / halves;
      *reinterpret_cast<uint16_t *>(p.out + r * p.pitch + (i - r * halves) * 2) = 0;
    }
  }
}

constexpr int kZeroThreads = 512;

// The zeros of a large dense gradient, most of its bytes.  The sort needs few
// SMs and waits for memory most of the time, so it runs at the same time: every
// CTA here lets it start once the kernels before this one are complete, and the
// sort waits for this kernel before it ends.
__global__ void __launch_bounds__(kZeroThreads) embedding_zero_kernel(const ZeroParams p) {
  ptx::grid_wait_prerequisites();
  ptx::grid_launch_dependents();
  write_zeros(p, static_cast<int64_t>(blockIdx.x) * kZeroThreads + threadIdx.x,
              static_cast<int64_t>(gridDim.x) * kZeroThreads);
}

// Inclusive sum over the warp's lanes.
__device__ __forceinline__ unsigned warp_scan(unsigned v) {
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const unsigned u = __shfl_up_sync(0xffffffffu, v, m);
    if ((threadIdx.x & 31) >= m) v += u;
  }
  return v;
}

// Lanes (of those in `among`) whose digits equal this one's, by eight votes: the
// match instruction takes longer the more different values the warp holds.
__device__ __forceinline__ unsigned equals(unsigned among, unsigned d) {
#pragma unroll
  for (int b = 0; b < 8; ++b) {
    const unsigned vote = __ballot_sync(0xffffffffu, (d >> b) & 1u);
    among &= (d >> b) & 1u ? vote : ~vote;
  }
  return among;
}
// Reads a word of another CTA's shared memory (of the same cluster).
__device__ __forceinline__ unsigned load_from_cta(const unsigned *p, int rank) {
  unsigned v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v)
               : "r"(ptx::mapa_shared(ptx::smem_u32(p), rank)) : "memory");
  return v;
}

// Stable least-significant-digit radix sort of (id, position), eight bits a
// pass.  Every warp owns a stretch of the list.  It counts its digits in order
// (lanes with equal digits find one another; the first adds them to the warp's
// own counter), which also ranks every token among the warp's equals; the
// counters of all warps and CTAs, summed by digit, CTA and warp, say where each
// goes.  With ITEMS > 0 a thread's tokens stay in registers between the two
// steps, all loads in flight together; ITEMS = 0 takes any number, reading
// them twice.
template <typename Id, int ITEMS>
__global__ void __launch_bounds__(kSortThreads) embedding_sort_kernel(const SortParams p) {
  constexpr int N = ITEMS > 0 ? ITEMS : 1;
  __shared__ alignas(16) unsigned s_cnt[kSortWarps][kDigits];
  __shared__ unsigned s_total[kDigits];  // of this CTA, read by the cluster
  __shared__ unsigned s_warp[kDigits / 32];
  // behind the zeros everything older is complete already
  if (!p.behind_zeros) ptx::grid_wait_prerequisites();
  const int rank = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (rank == 0 && tid < 2) p.count[tid] = 0;
  // this CTA's tokens, and this warp's part of them, in order
  const int b0 = static_cast<int>(static_cast<int64_t>(p.n) * rank / p.cluster);
  const int b1 = static_cast<int>(static_cast<int64_t>(p.n) * (rank + 1) / p.cluster);
  const int chunk = ((b1 - b0 + kSortThreads - 1) / kSortThreads) * 32;
  const int w0 = min(b1, b0 + warp * chunk), w1 = min(b1, w0 + chunk);
  const Id *ids = static_cast<const Id *>(p.ids);
  if (p.zeros.rows > 0)
    write_zeros(p.zeros, rank * kSortThreads + tid, p.cluster * kSortThreads);
  const unsigned below = (1u << lane) - 1;
  // a cluster of one CTA spares itself the wider barrier's fence
  const auto meet = [&] {
    if (p.cluster == 1) __syncthreads();
    else ptx::cluster_sync();
  };
  // adds the lanes `same` to their digit's counter; returns this lane's rank
  const auto tally = [&](unsigned same, bool on, unsigned d) {
    const unsigned at = on ? s_cnt[warp][d] + __popc(same & below) : 0u;
    __syncwarp();
    if (on && (same & below) == 0) s_cnt[warp][d] += __popc(same);
    __syncwarp();
    return at;
  };

  for (int pass = 0; pass < p.passes; ++pass) {
    const Entry *in = pass & 1 ? p.list0 : p.list1;
    Entry *out = pass & 1 ? p.list1 : p.list0;
    const int shift = 32 + 8 * pass;
    const auto load = [&](int i) {
      // from L2: what an SM may have cached is older than this kernel's start
      return pass ? __ldcg(in + i) : entry_of(key_of(__ldcg(ids + i), p), static_cast<unsigned>(i));
    };
    const auto digit = [&](Entry e) { return static_cast<unsigned>(e >> shift) & (kDigits - 1); };
    Entry item[N];
    unsigned at[N];
    if constexpr (ITEMS > 0) {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int i = w0 + k * 32 + lane;
        item[k] = i < w1 ? load(i) : 0;
      }
    }
#pragma unroll
    for (int i = tid; i < kSortWarps * kDigits / 4; i += kSortThreads)
      reinterpret_cast<uint4 *>(&s_cnt[0][0])[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    if constexpr (ITEMS > 0) {
#pragma unroll
      for (int k = 0; k < N; ++k)
        at[k] = equals(__ballot_sync(0xffffffffu, w0 + k * 32 + lane < w1), digit(item[k]));
#pragma unroll
      for (int k = 0; k < N; ++k) at[k] = tally(at[k], w0 + k * 32 + lane < w1, digit(item[k]));
    } else {
      for (int i = w0 + lane; i - lane < w1; i += 32) {
        const unsigned d = i < w1 ? digit(load(i)) : 0u;
        tally(equals(__ballot_sync(0xffffffffu, i < w1), d), i < w1, d);
      }
    }
    __syncthreads();
    // digit totals of the CTA, over the cluster
    if (tid < kDigits) {
      unsigned mine = 0;
#pragma unroll
      for (int w = 0; w < kSortWarps; ++w) mine += s_cnt[w][tid];
      s_total[tid] = mine;
    }
    meet();
    unsigned before = 0, total = 0, scan = 0;
    if (tid < kDigits) {
#pragma unroll
      for (int r = 0; r < kMostCluster; ++r) {
        const unsigned h = r < p.cluster ? load_from_cta(s_total + tid, r) : 0u;
        if (r < rank) before += h;
        total += h;
      }
      scan = warp_scan(total);
      if (lane == 31) s_warp[warp] = scan;
    }
    __syncthreads();
    if (tid < kDigits) {
      unsigned first = scan - total + before;
#pragma unroll
      for (int w = 0; w < kDigits / 32; ++w)
        if (w < warp) first += s_warp[w];
#pragma unroll
      for (int w = 0; w < kSortWarps; ++w) {
        const unsigned c = s_cnt[w][tid];
        s_cnt[w][tid] = first;
        first += c;
      }
    }
    __syncthreads();
    if constexpr (ITEMS > 0) {
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (w0 + k * 32 + lane < w1) out[s_cnt[warp][digit(item[k])] + at[k]] = item[k];
    } else {
      for (int i = w0 + lane; i - lane < w1; i += 32) {
        const Entry e = i < w1 ? load(i) : 0;
        const unsigned to =
            tally(equals(__ballot_sync(0xffffffffu, i < w1), digit(e)), i < w1, digit(e));
        if (i < w1) out[to] = e;
      }
    }
    // the next pass reads other CTAs' entries; no CTA leaves while its totals are read
    meet();
  }
  ptx::grid_launch_dependents();
  if (p.behind_zeros) ptx::grid_wait_prerequisites();
}

// -------------------------------------------------------------------- sums
struct SumParams {
  const void *dy;
  void *out;
  const Entry *list;
  // runs of equal ids that go on past the tile they begin in, as 2 * tile + slot
  // (slot 1: they begin further in than its first token): of at most kShort
  // pieces, and of more
  unsigned *count;   // [2]
  unsigned *owner0, *owner1;
  float *partial;    // [tile][2][pdim]: a run's piece at the tile's start, or further in
  int64_t dy_ld, out_ld;
  int n, rows, dim, pdim, slices;
  float scale;
  int accumulate;
};

// What the sums of VEC columns are added to, 16 bytes of the output at a time.
template <typename O, int VEC>
__device__ __forceinline__ void widen_old(const void *src, float (&old)[VEC]) {
  constexpr int P = VEC < vio::Full<O>::value ? VEC : vio::Full<O>::value;
#pragma unroll
  for (int k = 0; k < VEC; k += P) {
    float f[P];
    vio::unpack(vio::load_pack<O, P>(static_cast<const O *>(src) + k), f);
#pragma unroll
    for (int e = 0; e < P; ++e) old[k + e] = f[e];
  }
}
template <typename O>
__device__ __forceinline__ O *place_of(const SumParams &p, unsigned row, int c) {
  return static_cast<O *>(p.out) + static_cast<int64_t>(row) * p.out_ld + c;
}
// The finished sums.  (fp32 atomics in L2 would spare the old values' way here,
// but they flush subnormals to zero, and round twice.)
template <typename O, int VEC>
__device__ __forceinline__ void finish(const SumParams &p, unsigned row, int c,
                                       const float (&v)[VEC], const float (&old)[VEC]) {
  constexpr int P = VEC < vio::Full<O>::value ? VEC : vio::Full<O>::value;
  O *dst = place_of<O>(p, row, c);
#pragma unroll
  for (int k = 0; k < VEC; k += P) {
    float f[P];
#pragma unroll
    for (int e = 0; e < P; ++e) f[e] = fmaf(v[k + e], p.scale, old[k + e]);
    vio::store<O, P>(dst + k, f);
  }
}
template <typename O, int VEC>
__device__ __forceinline__ void finish(const SumParams &p, unsigned row, int c,
                                       const float (&v)[VEC]) {
  float old[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) old[e] = 0.f;
  if (p.accumulate) widen_old<O, VEC>(place_of<O>(p, row, c), old);
  finish<O, VEC>(p, row, c, v, old);
}

constexpr int kSumThreads = 256;
// Rows on their way per warp: every thread copies its part of them asynchronously
// into slots of its own in shared memory, so the loop over the tile's tokens is
// short and a warp waits for its next row only.  (Parts of two bytes, which
// cannot be copied so, are loaded kBatch rows and kWide columns at a time
// instead.)  The sums of 65536 tokens x 2048 columns of bf16, their 10000 fp32 rows
// left to atomics: 105 us with 16 rows and 3 CTAs per SM, 104 to 108 with 4 to 24
// rows and 8 to 2, and with batches of 16 rows in registers.
// Where the sums are added to existing rows, the row's old values travel with the
// last token of its run, and each slot holds both.  65536 x 2048 bf16 added to fp32
// 130 us with 4 slots, 131 with 8, 142 with 16 (of 8 columns a thread instead of 4:
// 145 with 8); 65536 x 512 fp32 62, 66, 71; old values loaded where a run ends: 133,
// 76.
template <bool ADD>
constexpr int kAhead = ADD ? 4 : 16;
constexpr int kBatch = 8, kWide = 4;

// Columns that a warp takes of a tile: 32 of VEC each, or kWide times 32 of two
// bytes.
template <typename T, int VEC>
constexpr int kSliceColumns = 32 * VEC * (sizeof(T) * VEC >= 4 ? 1 : kWide);

// Whether parts of VEC elements of T (and of O, where they are added to those) can
// be copied asynchronously, and the bytes of shared memory that a thread has for them.
template <typename T, int VEC>
constexpr bool kCopied = sizeof(T) * VEC >= 4;
template <typename T, typename O, int VEC, bool ADD>
constexpr int kRingBytes =
    kCopied<T, VEC> ? kAhead<ADD> * static_cast<int>(VEC * (sizeof(T) + (ADD ? sizeof(O) : 0))) : 0;

// One warp per (tile, slice of the columns).
template <typename T, typename O, int VEC, bool ADD>
__global__ void __launch_bounds__(kSumThreads, 3) embedding_sum_kernel(const SumParams p) {
  constexpr int kBytes = sizeof(T) * VEC;
  constexpr bool kAsync = kCopied<T, VEC>;
  constexpr int W = kAsync ? 1 : kWide;  // a thread's columns are c + 32 w (+ VEC)
  constexpr int kDepth = kAhead<ADD>;
  constexpr int kSlot = 32 * kBytes;
  constexpr int kOldBytes = sizeof(O) * VEC, kOldPart = kOldBytes < 16 ? kOldBytes : 16;
  // [warp][kDepth][lane] of dy, then of the old values (in parts of 16 bytes at most
  // [part][lane]), where copies are asynchronous
  extern __shared__ float4 s_dyn[];
  ptx::grid_launch_dependents();
  ptx::grid_wait_prerequisites();
  const int lane = threadIdx.x & 31;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * (kSumThreads / 32) + (threadIdx.x >> 5);
  const int64_t tile = item / p.slices;
  const int c = static_cast<int>(item - tile * p.slices) * kSliceColumns<T, VEC> + lane * VEC;
  const int64_t first = tile * kTile;
  if (first >= p.n) return;
  const Entry none = entry_of(static_cast<unsigned>(p.rows), 0);
  const Entry e = first + lane < p.n ? p.list[first + lane] : none;
  const unsigned before = key_in(first > 0 ? p.list[first - 1] : none);
  const unsigned after = key_in(first + kTile < p.n ? p.list[first + kTile] : none);
  const unsigned key = key_in(e), pos = static_cast<unsigned>(e);
  const int count = __popc(__ballot_sync(0xffffffffu, key != key_in(none)));  // rows come first
  const unsigned next = __shfl_down_sync(0xffffffffu, key, 1);
  // bit j: token j is the last of its run within the tile
  const unsigned ends = __ballot_sync(0xffffffffu, lane == 31 || key != next);
  // bit j: the run lies inside the tile and is finished here (equal ids are together)
  const unsigned closed = __ballot_sync(0xffffffffu, ((ends >> lane) & 1u) && key != before &&
                                                         (lane < kTile - 1 || key != after));
  const T *dy = static_cast<const T *>(p.dy) + c;
  const bool col = c < p.dim;
  char *ring = reinterpret_cast<char *>(s_dyn) + (threadIdx.x >> 5) * kDepth * kSlot + lane * kBytes;
  char *old_ring = reinterpret_cast<char *>(s_dyn) + kSumThreads / 32 * kDepth * kSlot +
                   (threadIdx.x >> 5) * kDepth * 32 * kOldBytes + lane * kOldPart;
  const auto row_of = [&](int t) {  // token t's row of dy, for the whole warp
    return dy + static_cast<int64_t>(__shfl_sync(0xffffffffu, pos, t & 31)) * p.dy_ld;
  };
  const auto fetch = [&](int t) {
    const T *src = row_of(t);
    if (col && t < count) vio::copy_async<kAsync ? kBytes : 4>(ring + t % kDepth * kSlot, src);
    if constexpr (ADD && kAsync) {
      const unsigned row = __shfl_sync(0xffffffffu, key, t & 31);
      if (col && t < count && ((closed >> t) & 1u)) {
#pragma unroll
        for (int k = 0; k < kOldBytes; k += kOldPart)
          vio::copy_async<kOldPart>(old_ring + t % kDepth * 32 * kOldBytes + k * 32,
                                    reinterpret_cast<const char *>(place_of<O>(p, row, c)) + k);
      }
    }
    vio::copy_commit();
  };
  if constexpr (kAsync) {
#pragma unroll 4
    for (int t = 0; t < kDepth; ++t) fetch(t);
  }
  float acc[W][VEC];
  const auto clear = [&] {
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[w][k] = 0.f;
  };
  clear();
  int begin = 0;
  vio::Pack<T, VEC> batch[kAsync ? 1 : kBatch][W];
#pragma unroll 1
  for (int t = 0; t < count; ++t) {
    if constexpr (!kAsync) {
      if (t % kBatch == 0) {
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          const T *src = row_of(t + j);
#pragma unroll
          for (int w = 0; w < W; ++w)
            if (c + 32 * w < p.dim && t + j < count)
              batch[j][w] = vio::load_pack<T, VEC>(src + 32 * w);
        }
      }
    } else {
      asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
      batch[0][0] = vio::load_pack<T, VEC>(ring + t % kDepth * kSlot);
    }
    float old[VEC];
    if constexpr (ADD && kAsync) {
      if ((closed >> t) & 1u) {
#pragma unroll
        for (int k = 0; k < kOldBytes; k += kOldPart) {
          constexpr int P = kOldPart / sizeof(O);
          float f[P];
          vio::unpack(vio::load_pack<O, P>(old_ring + t % kDepth * 32 * kOldBytes + k * 32), f);
#pragma unroll
          for (int e = 0; e < P; ++e) old[k / static_cast<int>(sizeof(O)) + e] = f[e];
        }
      }
    }
#pragma unroll
    for (int w = 0; w < W; ++w) {
      float v[VEC];
      vio::unpack(batch[0][w], v);
      if (c + 32 * w < p.dim) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[w][k] += v[k];
      }
#pragma unroll
      for (int j = 0; j + 1 < (kAsync ? 1 : kBatch); ++j) batch[j][w] = batch[j + 1][w];
    }
    if constexpr (kAsync) fetch(t + kDepth);
    if (!((ends >> t) & 1u)) continue;
    const unsigned row = __shfl_sync(0xffffffffu, key, t);
    const bool goes_on = t == kTile - 1 && after == row;
    const bool open = !((closed >> t) & 1u);
    if (goes_on && !(begin == 0 && before == row) && c == 0) {
      // where the run still is if it has more pieces; the lists' order changes nothing
      const int64_t far = first + int64_t(kShort) * kTile;
      const bool is_long = far < p.n && key_in(p.list[far]) == row;
      const unsigned at = atomicAdd(p.count + (is_long ? 1 : 0), 1u);
      (is_long ? p.owner1 : p.owner0)[at] = static_cast<unsigned>(2 * tile + (begin ? 1 : 0));
    }
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const int cw = c + 32 * w;
      if (cw >= p.dim) continue;
      if (open) {
        float *dst = p.partial + (tile * 2 + (begin ? 1 : 0)) * p.pdim + cw;
        if constexpr (VEC % 4 == 0) {
#pragma unroll
          for (int k = 0; k < VEC; k += 4)
            __stcg(reinterpret_cast<float4 *>(dst + k),
                   make_float4(acc[w][k], acc[w][k + 1], acc[w][k + 2], acc[w][k + 3]));
        } else {
#pragma unroll
          for (int k = 0; k < VEC; ++k) __stcg(dst + k, acc[w][k]);
        }
      } else if constexpr (ADD && kAsync) {
        finish<O, VEC>(p, row, cw, acc[w], old);
      } else {
        finish<O, VEC>(p, row, cw, acc[w]);
      }
    }
    clear();
    begin = t + 1;
  }
}

// Writes four columns of a joined run.
template <typename O>
__device__ __forceinline__ void finish_four(const SumParams &p, unsigned row, int c, float4 s,
                                            bool vectors) {
  const float f[4] = {s.x, s.y, s.z, s.w};
  if (vectors) {
    if (c < p.dim) finish<O, 4>(p, row, c, f);
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float one[1] = {f[k]};
    if (c + k < p.dim) finish<O, 1>(p, row, c + k, one);
  }
}
__device__ __forceinline__ void add4(float4 *s, const float4 v) {
  s->x += v.x;
  s->y += v.y;
  s->z += v.z;
  s->w += v.w;
}

// Runs that cross tiles, 128 columns at a time.  A warp joins a run of few
// pieces, all loads in flight; a CTA one of many, each warp a stretch of them in
// order and then the warps' sums in order.
template <typename O>
__global__ void __launch_bounds__(kSumThreads) embedding_join_kernel(const SumParams p,
                                                                     const int vectors) {
  constexpr int kWarps = kSumThreads / 32;
  __shared__ float4 s_sum[kWarps][32];
  ptx::grid_launch_dependents();
  ptx::grid_wait_prerequisites();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int slices = (p.pdim + 127) / 128;
  const int64_t few = static_cast<int64_t>(p.count[0]) * slices;
  const int64_t many = static_cast<int64_t>(p.count[1]) * slices;
  for (int64_t item = blockIdx.x; item < many; item += gridDim.x) {
    const unsigned o = p.owner1[item / slices];
    const int c = static_cast<int>(item % slices) * 128 + lane * 4;
    const int64_t tile = o >> 1;
    const unsigned row = key_in(p.list[tile * kTile + kTile - 1]);
    // tiles after this one whose first token is still of the run
    int more = kShort;
    for (;;) {
      const int64_t t = (tile + 1 + more + lane) * kTile;
      const unsigned on = __ballot_sync(0xffffffffu, t < p.n && key_in(p.list[t]) == row);
      const int run = on == 0xffffffffu ? 32 : __ffs(~on) - 1;
      more += run;
      if (run < 32) break;
    }
    const int pieces = more + 1;
    const int per = (pieces + kWarps - 1) / kWarps;
    const int a = min(pieces, warp * per), b = min(pieces, a + per);
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (c < p.pdim) {
#pragma unroll 8
      for (int k = a; k < b; ++k) {
        const int64_t at = (tile + k) * 2 + (k == 0 ? o & 1 : 0u);
        add4(&s, __ldcg(reinterpret_cast<const float4 *>(p.partial + at * p.pdim + c)));
      }
    }
    s_sum[warp][lane] = s;
    __syncthreads();
    if (warp == 0) {
      for (int w = 1; w < kWarps; ++w) add4(&s, s_sum[w][lane]);
      finish_four<O>(p, row, c, s, vectors != 0);
    }
    __syncthreads();
  }
  for (int64_t item = static_cast<int64_t>(blockIdx.x) * kWarps + warp; item < few;
       item += static_cast<int64_t>(gridDim.x) * kWarps) {
    const unsigned o = p.owner0[item / slices];
    const int c = static_cast<int>(item % slices) * 128 + lane * 4;
    const int64_t tile = o >> 1;
    // lane k >= 1: whether the run still is at tile + k; the row from lane 0
    const int64_t t = lane == 0 ? tile * kTile + kTile - 1 : (tile + lane) * kTile;
    const unsigned key = lane < kShort && t < p.n ? key_in(p.list[t]) : ~0u;
    const unsigned row = __shfl_sync(0xffffffffu, key, 0);
    const int pieces = __ffs(~__ballot_sync(0xffffffffu, key == row)) - 1;
    if (c >= p.pdim) continue;
    float4 v[kShort], s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < kShort; ++k) {
      const int64_t at = (tile + k) * 2 + (k == 0 ? o & 1 : 0u);
      if (k < pieces) v[k] = __ldcg(reinterpret_cast<const float4 *>(p.partial + at * p.pdim + c));
    }
#pragma unroll
    for (int k = 0; k < kShort; ++k)
      if (k < pieces) add4(&s, v[k]);
    finish_four<O>(p, row, c, s, vectors != 0);
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
  // 8 CTAs per SM that loop: 62 us for 65536 rows of 4 KB, against 67 with 64 per SM and
  // 73 with a CTA for every four rows
  const int grid = static_cast<int>(std::min<int64_t>(want, int64_t(8) * device_info(dev).sm_count));
  return launched(wide_ids ? launch_dependent(embedding_forward_kernel<T, int64_t, VEC>, dim3(grid),
                                              dim3(kLookThreads), 0, stream, p)
                           : launch_dependent(embedding_forward_kernel<T, int32_t, VEC>, dim3(grid),
                                              dim3(kLookThreads), 0, stream, p),
                  "embedding_forward_kernel");
}

template <typename T, int VEC = vio::Full<T>::value>
int look_any(const LookParams &p, bool wide_ids, cudaStream_t stream) {
  const bool fits = p.dim % VEC == 0 && p.ld % VEC == 0 && aligned(p.table, VEC * sizeof(T)) &&
                    aligned(p.out, VEC * sizeof(T));
  if constexpr (VEC > 1) {
    if (!fits) return look_any<T, VEC / 2>(p, wide_ids, stream);
  }
  return look<T, VEC>(p, wide_ids, stream);
}

struct Layout {  // of the backward's workspace
  size_t list[2], count, owner[2], partial, bytes;
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
    l.list[i] = take(n * sizeof(Entry));
    l.owner[i] = take(sizeof(unsigned) * static_cast<size_t>(l.tiles));
  }
  l.count = take(2 * sizeof(unsigned));
  l.partial = take(sizeof(float) * 2 * static_cast<size_t>(l.tiles) * l.pdim);
  l.bytes = at;
  return l;
}

template <typename Id, int ITEMS>
void sort_config(cudaLaunchConfig_t *cfg, cudaLaunchAttribute (&attr)[2], int cluster) {
  *cfg = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg->gridDim = dim3(cluster);
  cfg->blockDim = dim3(kSortThreads);
  cfg->attrs = attr;
  cfg->numAttrs = 1;
}

template <typename Id, int ITEMS>
int sort_ids(SortParams p, int cluster, cudaStream_t stream) {
  auto kernel = embedding_sort_kernel<Id, ITEMS>;
  p.cluster = cluster;
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr[2];
  sort_config<Id, ITEMS>(&cfg, attr, cluster);
  if (cluster > 8) {
    static thread_local int seen_device = -1;
    const int dev = current_device();
    if (seen_device != dev) {
      const cudaError_t e =
          cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      if (e != cudaSuccess) return launched(e, "embedding_sort_kernel");
      seen_device = dev;
    }
  }
  cfg.stream = stream;
  cfg.numAttrs = programmatic_launch_enabled() ? 2 : 1;
  return launched(cudaLaunchKernelEx(&cfg, kernel, p), "embedding_sort_kernel");
}

// The largest sorting cluster of the current device: 16 CTAs where one of that
// size fits, else the 8 that every device takes (0 on an error).
int most_sorting_ctas() {
  static thread_local int seen_device = -1, most = 8;
  const int dev = current_device();
  if (dev < 0) return 0;
  if (seen_device == dev) return most;
  auto kernel = embedding_sort_kernel<int64_t, 8>;
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr[2];
  sort_config<int64_t, 8>(&cfg, attr, kMostCluster);
  int fits = 0;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) !=
          cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&fits, kernel, &cfg) != cudaSuccess) {
    (void)cudaGetLastError();
    fits = 0;
  }
  most = fits > 0 ? kMostCluster : 8;
  seen_device = dev;
  return most;
}

// One CTA takes up to 2048 tokens (8.2 us for two passes of 2000; two CTAs 8.7,
// but four CTAs 9.0 and one 12.7 for 4000), then a token a thread up to the
// largest cluster, then 2, 4 or 8 a thread in registers (8 spill 48 bytes), then any
// number.
constexpr int kOneCta = 2 * kSortThreads;
template <typename Id>
int sort_any(const SortParams &p, cudaStream_t stream) {
  const int most = most_sorting_ctas();
  if (most == 0) return fail(BEVK_ERR_CUDA, "embedding_backward: no device");
  int cluster = 1;
  while (p.n > kOneCta && cluster < most && p.n > kSortThreads * cluster) cluster *= 2;
  const int each = (p.n + cluster - 1) / cluster;
  if (each <= kSortThreads) return sort_ids<Id, 1>(p, cluster, stream);
  if (each <= 2 * kSortThreads) return sort_ids<Id, 2>(p, cluster, stream);
  if (each <= 4 * kSortThreads) return sort_ids<Id, 4>(p, cluster, stream);
  if (each <= 8 * kSortThreads) return sort_ids<Id, 8>(p, cluster, stream);
  return sort_ids<Id, 0>(p, cluster, stream);
}

template <typename T, typename O, int VEC, bool ADD>
int sum(const SumParams &p0, int64_t tiles, cudaStream_t stream) {
  SumParams p = p0;
  p.slices = (p.dim + kSliceColumns<T, VEC> - 1) / kSliceColumns<T, VEC>;
  const int64_t warps = tiles * p.slices, per = kSumThreads / 32;
  const int64_t grid = (warps + per - 1) / per;
  if (grid >= (int64_t(1) << 31))
    return fail(BEVK_ERR_INDEX_OVERFLOW, "embedding_backward: too many tokens and columns");
  const size_t smem = static_cast<size_t>(kRingBytes<T, O, VEC, ADD>) * kSumThreads;
  if (smem > 0) {
    static thread_local int seen_device = -1;
    const int dev = current_device();
    if (dev < 0) return fail(BEVK_ERR_CUDA, "embedding_backward: no device");
    if (seen_device != dev) {
      const cudaError_t e = cudaFuncSetAttribute(embedding_sum_kernel<T, O, VEC, ADD>,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 static_cast<int>(smem));
      if (e != cudaSuccess) return launched(e, "embedding_sum_kernel");
      seen_device = dev;
    }
  }
  const int st = launched(launch_dependent(embedding_sum_kernel<T, O, VEC, ADD>,
                                           dim3(static_cast<unsigned>(grid)), dim3(kSumThreads),
                                           smem, stream, p),
                          "embedding_sum_kernel");
  if (st != BEVK_OK) return st;
  if (tiles < 2) return BEVK_OK;  // no run crosses tiles
  const int64_t items = (tiles - 1) * ((p.pdim + 127) / 128);
  const int64_t most = int64_t(8) * device_info(current_device()).sm_count;
  const int vectors = p.dim % 4 == 0 && p.out_ld * sizeof(O) % 16 == 0 && aligned(p.out, 16);
  return launched(launch_dependent(embedding_join_kernel<O>,
                                   dim3(static_cast<unsigned>(std::min(items, most))),
                                   dim3(kSumThreads), 0, stream, p, vectors),
                  "embedding_join_kernel");
}

// The widest part of a row, up to 16 bytes of dy (of the wider side where both are
// copied), that every row's start and length are a multiple of on the side of dy, and
// its columns on the side of the table.
template <typename T, typename O, bool ADD, int VEC = vio::Full<std::conditional_t<ADD, O, T>>::value>
int sum_any(const SumParams &p, int64_t tiles, cudaStream_t stream) {
  constexpr size_t kOut = std::min<size_t>(16, VEC * sizeof(O));
  const bool fits = p.dim % VEC == 0 && p.dy_ld % VEC == 0 && aligned(p.dy, VEC * sizeof(T)) &&
                    p.out_ld * sizeof(O) % kOut == 0 && aligned(p.out, kOut);
  if constexpr (VEC > 1) {
    if (!fits) return sum_any<T, O, ADD, VEC / 2>(p, tiles, stream);
  }
  return sum<T, O, VEC, ADD>(p, tiles, stream);
}
template <typename T, typename O>
int sum_any(const SumParams &p, int64_t tiles, cudaStream_t stream) {
  return p.accumulate ? sum_any<T, O, true>(p, tiles, stream)
                      : sum_any<T, O, false>(p, tiles, stream);
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
  s.list0 = reinterpret_cast<Entry *>(base + l.list[0]);
  s.list1 = reinterpret_cast<Entry *>(base + l.list[1]);
  s.count = reinterpret_cast<unsigned *>(base + l.count);
  s.rows = a->num_rows;
  s.padding = a->padding_idx;
  s.n = static_cast<int>(a->num_ids);
  s.passes = 1;
  while (s.passes < 4 && (a->num_rows >> (8 * s.passes)) != 0) ++s.passes;
  int st = BEVK_OK;
  if (!a->accumulate) {
    const int64_t size = dtype_size(a->grad_table_dtype);
    const ZeroParams z = {static_cast<char *>(grad_table), a->num_rows, a->dim * size,
                          a->grad_table_ld * size};
    const int64_t bytes = z.rows * z.row_bytes;
    // four stores of every sorting thread cost less than a launch
    const int64_t few = std::max<int64_t>(1, std::min<int64_t>(8, s.n / kSortThreads)) *
                        kSortThreads * 64;
    if (bytes <= few) {
      s.zeros = z;
    } else {
      const int64_t want = (bytes + 64 * kZeroThreads - 1) / (64 * kZeroThreads);
      const int dev = current_device();
      if (dev < 0) return fail(BEVK_ERR_CUDA, "embedding_backward: no device");
      const int64_t most = int64_t(2) * device_info(dev).sm_count;  // leaves the sort room
      st = launched(launch_dependent(embedding_zero_kernel,
                                     dim3(static_cast<unsigned>(std::min(want, most))),
                                     dim3(kZeroThreads), 0, stream, z),
                    "embedding_zero_kernel");
      if (st != BEVK_OK) return st;
      s.behind_zeros = programmatic_launch_enabled();
    }
  }
  st = a->ids_are_64bit ? sort_any<int64_t>(s, stream) : sort_any<int32_t>(s, stream);
  if (st != BEVK_OK) return st;
  SumParams p = {};
  p.dy = dy;
  p.out = grad_table;
  p.list = s.passes & 1 ? s.list0 : s.list1;
  p.count = s.count;
  p.owner0 = reinterpret_cast<unsigned *>(base + l.owner[0]);
  p.owner1 = reinterpret_cast<unsigned *>(base + l.owner[1]);
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
