// Embedding lookup with scaling, and the gradient of its table by sorted tokens: what the adapters' trunk begins with
// (adapters/mlx_lm.py:140-164 of the reference calls the model's own embedding module).
//
// Forward: y_i = scale W[id_i], a read and a write of N rows.  Backward: dW[v] = scale sum of dy_i over the i with id_i = v, held in
// fp32 and rounded once; it reads N rows and writes all V rows, nearly all of them zero, so the writes bound it.  The order
// of a sum is fixed (token by token in a window, windows in turn) and there are no atomics, so equal calls give equal bits:
//   1. one cluster sorts the tokens by id (stable, least digits first); beside it a second kernel fills the table with zeros, so that
//      the sort's dependent steps cost nothing where the table is large (V = 151936, D = 4096: 170 us of writes at 7.3 TB/s);
//   2. windows of the sorted tokens sum the rows of each run of equal ids; a run that lies in one window is written, one that
//      crosses a border leaves a partial sum;
//   3. the partial sums of runs that cross borders are joined in order.  A padding id that fills half a batch is thousands
//      of rows: step 2 spreads them over all SMs, and one CTA for 256 columns adds up what is left of them.
//
// Up to 64 tokens need no sort: one kernel fills the table, and a CTA that finds ids among its rows sums those as well.  Forward and
// backward on the device, 32768 x 2048 bf16: 16 tokens 23 us against 27, 64 tokens 26 against 28, and one launch in place
// of four (12 us of host time, of some 100).  That CTA's reads wait behind all others' writes: 54 equal ids of 64 take 44 us
// against 28, 150 of 250 would take 96 against 30.
//
// An id outside [0, V) gives a row of zeros, no gradient, and a status word.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "common.h"
#include "ptx.cuh"

namespace b200tp {
namespace {

namespace cg = cooperative_groups;

constexpr int kCluster = 8;
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kKeys = 4;                           // keys of a lane in flight
constexpr int kMaxDigit = 9;                       // bits of a sort's digit: 32 warps x 512 counters are 64 kB
constexpr long long kFillBytes = 64 << 10;         // of one CTA (256 kB: 172 us, 1 MB: 181 us for 1.24 GB)
constexpr int kCols = 8;                           // columns of a thread
constexpr int kThreads = 256;
constexpr int kSlice = kThreads * kCols;           // columns of a CTA that sums
constexpr int kJoinSlice = 256;                    // columns of a CTA that joins

__device__ __forceinline__ float value(float x) { return x; }
__device__ __forceinline__ float value(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// An id outside the table; a word that is already there stays.
__device__ __forceinline__ void report(int* status) {
  if (status != nullptr) atomicCAS(status, 0, B200TP_DEV_BAD_INDEX);
}

// Eight columns of a row.  VEC: adjacent ones from `col`, 16-byte loads; else `col + j * step`, those below d.
template <typename T, bool VEC>
struct Cols {
  uint4 raw[VEC ? sizeof(T) / 2 : 1];
  T one[VEC ? 1 : kCols];

  __device__ __forceinline__ void load(const T* row, int col, int step, int d) {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
        raw[i] = col < d ? __ldg(reinterpret_cast<const uint4*>(row + col) + i) : make_uint4(0, 0, 0, 0);
    } else {
#pragma unroll
      for (int j = 0; j < kCols; ++j) one[j] = col + j * step < d ? row[col + j * step] : T(0.f);
    }
  }
  __device__ __forceinline__ void add_to(float (&acc)[kCols]) const {
    float v[kCols];
    get(v);
#pragma unroll
    for (int j = 0; j < kCols; ++j) acc[j] += v[j];
  }
  __device__ __forceinline__ void get(float (&v)[kCols]) const {
    if constexpr (!VEC) {
#pragma unroll
      for (int j = 0; j < kCols; ++j) v[j] = value(one[j]);
    } else if constexpr (sizeof(T) == 2) {
      const uint32_t w[4] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = __uint_as_float(w[j] << 16);
        v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
      }
    } else {
      const uint4 a = raw[0], b = raw[1];
      const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(w[j]);
    }
  }
};

template <typename T, bool VEC>
__device__ __forceinline__ void store_cols(T* row, int col, int step, int d, const float (&v)[kCols], float scale) {
  if constexpr (!VEC) {
#pragma unroll
    for (int j = 0; j < kCols; ++j)
      if (col + j * step < d) put(row + col + j * step, v[j] * scale);
  } else if (col < d) {
    if constexpr (sizeof(T) == 2) {
      uint4 u;
      __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
      for (int j = 0; j < 4; ++j) h[j] = __floats2bfloat162_rn(v[2 * j] * scale, v[2 * j + 1] * scale);
      *reinterpret_cast<uint4*>(row + col) = u;
    } else {
      *reinterpret_cast<float4*>(row + col) = make_float4(v[0] * scale, v[1] * scale, v[2] * scale, v[3] * scale);
      *(reinterpret_cast<float4*>(row + col) + 1) = make_float4(v[4] * scale, v[5] * scale, v[6] * scale, v[7] * scale);
    }
  }
}

// A warp takes 4 x 256 columns of one row (VEC: four loads of 16 bytes or more in flight for each lane).
template <typename T, typename ID, bool VEC>
__global__ void __launch_bounds__(kThreads)
embed_fwd_kernel(const ID* __restrict__ ids, const T* __restrict__ weight, long long w_stride, long long n, int d, int parts,
                 long long v, float scale, T* __restrict__ out, int* status) {
  griddep_wait();
  griddep_launch_dependents();
  const long long item = static_cast<long long>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const long long row = item / parts;
  if (row >= n) return;
  const int first = static_cast<int>(item - row * parts) * 1024;
  const long long id = static_cast<long long>(ids[row]);
  const bool ok = id >= 0 && id < v;
  if (!ok && lane == 0) report(status);
  const T* from = weight + (ok ? id : 0) * w_stride;
  T* to = out + row * d;
  Cols<T, VEC> c[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) c[k].load(from, VEC ? first + (k * 32 + lane) * kCols : first + k * 256 + lane, 32, ok ? d : 0);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    float x[kCols];
    c[k].get(x);
    store_cols<T, VEC>(to, VEC ? first + (k * 32 + lane) * kCols : first + k * 256 + lane, 32, d, x, scale);
  }
}

constexpr int kDirect = 64;                        // tokens that are looked through by every CTA
constexpr int kDirectThreads = 512;

// Zeros over `rows` rows of the table, and the sums of those that have tokens: the CTA's threads look at all ids, and where some fall
// among its rows, each such row is summed over its tokens in their order, eight columns to a thread.
template <typename T, typename ID, bool VEC>
__global__ void __launch_bounds__(kDirectThreads)
embed_direct_kernel(const ID* __restrict__ ids, int n, long long v, long long padding, int rows, const T* __restrict__ dy,
                    long long dy_stride, int d, float scale, T* __restrict__ dw, int* status) {
  griddep_wait();
  griddep_launch_dependents();
  __shared__ int local[kDirect];                   // a token's row among the CTA's, or -1
  __shared__ unsigned match[kDirect / 32];
  const long long first = static_cast<long long>(blockIdx.x) * rows;
  const long long end = min(first + rows, v);
  const long long id = static_cast<int>(threadIdx.x) < n ? static_cast<long long>(ids[threadIdx.x]) : -1;    // n <= kDirect
  // rows are a multiple of eight, so that the CTA's share begins on a 16-byte boundary; the id arrives meanwhile
  const long long bytes = (end - first) * d * static_cast<long long>(sizeof(T));
  uint4* fill = reinterpret_cast<uint4*>(dw + first * d);
  for (long long i = threadIdx.x; i < bytes / 16; i += kDirectThreads) fill[i] = make_uint4(0, 0, 0, 0);
  if (threadIdx.x < (bytes & 15) / 2) reinterpret_cast<unsigned short*>(fill)[bytes / 16 * 8 + threadIdx.x] = 0;
  if (static_cast<int>(threadIdx.x) < n && (id < 0 || id >= v) && blockIdx.x == 0) report(status);
  const bool mine = id >= first && id < end && id != padding;
  if (threadIdx.x < kDirect) local[threadIdx.x] = mine ? static_cast<int>(id - first) : -1;
  if (!__syncthreads_or(mine)) return;             // the barrier also puts the zeros before the sums
  for (int t = 0; t < n; ++t) {
    const int row = local[t];
    if (row < 0) continue;                         // the same for all threads
    bool same = false;
    if (threadIdx.x < kDirect) {
      same = local[threadIdx.x] == row;
      const unsigned m = __ballot_sync(0xffffffffu, same);
      if ((threadIdx.x & 31) == 0) match[threadIdx.x >> 5] = m;
    }
    if (__syncthreads_or(same && static_cast<int>(threadIdx.x) < t)) continue;    // an earlier token had this row
    for (int base = 0; base < d; base += kDirectThreads * kCols) {
      const int col = base + (VEC ? threadIdx.x * kCols : threadIdx.x);
      if (col >= d) break;
      float acc[kCols] = {};
      constexpr int kAhead = 4;
      int word = t >> 5;
      unsigned left = match[word];
      bool more = true;
      while (more) {
        Cols<T, VEC> c[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          while (left == 0 && word + 1 < kDirect / 32) left = match[++word];
          more = left != 0;
          const int at = more ? word * 32 + __ffs(left) - 1 : 0;
          left &= left - 1;
          c[k].load(dy + at * dy_stride, col, kDirectThreads, more ? d : 0);     // nothing left: zeros
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) c[k].add_to(acc);
      }
      store_cols<T, VEC>(dw + (first + row) * d, col, kDirectThreads, d, acc, scale);
    }
    __syncthreads();                               // `match` is written again
  }
}

struct Sort {
  unsigned *key_a, *pos_a, *key_b, *pos_b;   // of n entries each: passes write a, b, a, ...
  long long n;
  long long v;                               // keys: ids in [0, v), and v for tokens without a gradient
  long long padding;                         // an id without a gradient, or -1
  int digit, passes;
};

// Zeros over the table, while the sort before it in the stream runs: nothing here waits for that one's results.  Whatever came
// before the sort is over (the sort lets this kernel start only after its own wait), and what comes after this one finds the sort
// finished because the last CTA here does not end before it.
__global__ void __launch_bounds__(kSortThreads) embed_fill_kernel(uint4* __restrict__ fill, long long bytes) {
  griddep_launch_dependents();
  const long long from = blockIdx.x * (kFillBytes / 16), to = min(from + kFillBytes / 16, bytes / 16);
  for (long long i = from + threadIdx.x; i < to; i += kSortThreads) fill[i] = make_uint4(0, 0, 0, 0);
  if (blockIdx.x == gridDim.x - 1) {
    if (threadIdx.x < (bytes & 15) / 2)                            // elements are of 2 or 4 bytes
      reinterpret_cast<unsigned short*>(fill)[bytes / 16 * 8 + threadIdx.x] = 0;
    griddep_wait();
  }
}

template <typename ID>
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kSortThreads)
embed_sort_kernel(const ID* __restrict__ ids, const Sort s, int* status) {
  griddep_wait();
  griddep_launch_dependents();
  cg::cluster_group cluster = cg::this_cluster();
  extern __shared__ unsigned shared[];
  const int bins = 1 << s.digit;
  unsigned* counts = shared;                 // [warp][bin]: tokens of this digit before the warp's next one, in this CTA
  unsigned* totals = counts + kSortWarps * bins;   // [bin]: of this CTA
  unsigned* bases = totals + bins;           // [bin]: place of this CTA's first token of this digit
  __shared__ unsigned sums[kSortWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster.block_rank());
  // a warp's tokens are adjacent, so that an order by (digit, warp, place) is stable
  const long long per = ((s.n + kCluster * kSortWarps - 1) / (kCluster * kSortWarps) + 31) / 32 * 32;
  const long long lo = min((rank * kSortWarps + warp) * per, s.n), hi = min(lo + per, s.n);
  unsigned* mine = counts + warp * bins;
  const unsigned none = 0xffffffffu;

  for (int pass = 0; pass < s.passes; ++pass) {
    const unsigned* key_in = pass & 1 ? s.key_a : s.key_b;
    const unsigned* pos_in = pass & 1 ? s.pos_a : s.pos_b;
    unsigned* key_out = pass & 1 ? s.key_b : s.key_a;
    unsigned* pos_out = pass & 1 ? s.pos_b : s.pos_a;
    const int shift = pass * s.digit;
    auto key_at = [&](long long i) -> unsigned {
      if (pass > 0) return __ldcg(key_in + i);                    // written by other CTAs of the cluster
      const long long id = static_cast<long long>(ids[i]);
      if (id >= 0 && id < s.v) return static_cast<unsigned>(id == s.padding ? s.v : id);
      report(status);
      return static_cast<unsigned>(s.v);
    };
    for (int b = threadIdx.x; b < kSortWarps * bins; b += kSortThreads) counts[b] = 0;
    __syncthreads();
    for (long long base = lo; base < hi; base += 32 * kKeys) {
      unsigned key[kKeys];
#pragma unroll
      for (int k = 0; k < kKeys; ++k) key[k] = base + k * 32 + lane < hi ? key_at(base + k * 32 + lane) : 0;
#pragma unroll
      for (int k = 0; k < kKeys; ++k) {                            // whole warps; lanes past the end have a digit of their own
        const bool in = base + k * 32 + lane < hi;
        const unsigned digit = in ? (key[k] >> shift) & (bins - 1) : none;
        const unsigned peers = __match_any_sync(0xffffffffu, digit);
        if (in && lane == __ffs(peers) - 1) mine[digit] += __popc(peers);
        __syncwarp();
      }
    }
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += kSortThreads) {      // counts -> tokens of this digit in warps before; totals
      unsigned run = 0;
#pragma unroll 8
      for (int w = 0; w < kSortWarps; ++w) {
        const unsigned c = counts[w * bins + b];
        counts[w * bins + b] = run;
        run += c;
      }
      totals[b] = run;
    }
    cluster.sync();
    unsigned before = 0, all = 0;                                  // bins <= kSortThreads: one bin a thread
    if (threadIdx.x < bins) {
#pragma unroll
      for (int r = 0; r < kCluster; ++r) {
        const unsigned c = cluster.map_shared_rank(totals, r)[threadIdx.x];
        all += c;
        if (r < rank) before += c;
      }
    }
    unsigned scan = all;                                           // sum over bins up to this one
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned up = __shfl_up_sync(0xffffffffu, scan, o);
      if (lane >= o) scan += up;
    }
    if (lane == 31) sums[warp] = scan;
    __syncthreads();
    unsigned below = 0;
    for (int w = 0; w < warp; ++w) below += sums[w];
    if (threadIdx.x < bins) bases[threadIdx.x] = below + scan - all + before;
    __syncthreads();
    for (long long base = lo; base < hi; base += 32 * kKeys) {
      unsigned key[kKeys], pos[kKeys];
#pragma unroll
      for (int k = 0; k < kKeys; ++k) {
        const long long i = base + k * 32 + lane;
        key[k] = i < hi ? key_at(i) : 0;
        pos[k] = i < hi && pass > 0 ? __ldcg(pos_in + i) : static_cast<unsigned>(i);
      }
#pragma unroll
      for (int k = 0; k < kKeys; ++k) {
        const bool in = base + k * 32 + lane < hi;
        const unsigned digit = in ? (key[k] >> shift) & (bins - 1) : none;
        const unsigned peers = __match_any_sync(0xffffffffu, digit);
        const unsigned at = in ? bases[digit] + mine[digit] + __popc(peers & ((1u << lane) - 1)) : 0;
        __syncwarp();
        if (in && lane == __ffs(peers) - 1) mine[digit] += __popc(peers);
        __syncwarp();
        if (in) {
          key_out[at] = key[k];
          pos_out[at] = pos[k];
        }
      }
    }
    __threadfence();
    cluster.sync();                                                // the next pass reads what all eight wrote, and counts anew
  }
}

// One window of sorted tokens and 2048 columns to a CTA.  Runs that end or begin outside the window leave their sum in `head` (they
// began before it) or `tail` (they begin in it and go on).
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads)
embed_sum_kernel(const unsigned* __restrict__ keys, const unsigned* __restrict__ pos, long long n, int window, long long v,
                 const T* __restrict__ dy, long long dy_stride, int d, float scale, T* __restrict__ dw, float* __restrict__ head,
                 float* __restrict__ tail) {
  griddep_wait();
  griddep_launch_dependents();
  constexpr int kMost = 64;
  __shared__ unsigned key_s[kMost + 2], pos_s[kMost];
  const long long first = static_cast<long long>(blockIdx.x) * window;
  const int count = static_cast<int>(min(static_cast<long long>(window), n - first));
  const unsigned none = 0xffffffffu;                               // no key: ids stop below 2^31
  for (int i = threadIdx.x; i < count + 2; i += kThreads) {
    const long long at = first + i - 1;
    key_s[i] = at >= 0 && at < n ? keys[at] : none;
    if (i >= 1 && i <= count) pos_s[i - 1] = pos[at];
  }
  __syncthreads();
  const int col = blockIdx.y * kSlice + (VEC ? threadIdx.x * kCols : threadIdx.x);
  if (col >= d) return;
  constexpr int kAhead = VEC && sizeof(T) == 2 ? 8 : 4;            // rows in flight
  float acc[kCols] = {};
  bool from_before = key_s[1] == key_s[0];
  for (int base = 0; base < count; base += kAhead) {
    Cols<T, VEC> c[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const bool use = base + k < count && key_s[base + k + 1] < v;
      c[k].load(dy + static_cast<long long>(use ? pos_s[base + k] : 0) * dy_stride, col, kThreads, use ? d : 0);
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = base + k;
      if (i >= count) break;
      const unsigned key = key_s[i + 1];
      if (key >= v) return;                                        // tokens without a gradient are the last ones
      c[k].add_to(acc);
      const bool goes_on = key_s[i + 2] == key;
      if (goes_on && i + 1 < count) continue;
      if (goes_on || from_before) {
        float* to = (from_before ? head : tail) + static_cast<long long>(blockIdx.x) * d;
        store_cols<float, VEC>(to, col, kThreads, d, acc, 1.f);
      } else {
        store_cols<T, VEC>(dw + key * static_cast<long long>(d), col, kThreads, d, acc, scale);
      }
      from_before = false;
#pragma unroll
      for (int j = 0; j < kCols; ++j) acc[j] = 0.f;
    }
  }
}

// Runs that begin in a window and go on: tail of that window, then heads of the windows up to the run's end.  A CTA takes 256
// columns, four to a thread; its four groups of 64 threads share the run's windows, and their sums are added in order.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads)
embed_join_kernel(const unsigned* __restrict__ keys, long long n, int window, long long v, int d, float scale,
                  const float* __restrict__ head, const float* __restrict__ tail, T* __restrict__ dw) {
  griddep_wait();
  griddep_launch_dependents();
  const long long w = blockIdx.x, first = w * window, next = first + window;
  if (next >= n) return;
  const unsigned key = keys[next - 1];
  if (key >= v || keys[next] != key) return;                       // no run goes on
  if (keys[first] == key && w > 0 && keys[first - 1] == key) return;   // it began before
  // The last window that the run reaches: each thread asks one window whether the run goes on behind it.
  __shared__ int stop;
  long long last = w + 1;
  for (;; last += kThreads) {
    const long long end = (last + threadIdx.x + 1) * window;       // first token behind the window
    const bool goes_on = end < n && keys[end - 1] == key && keys[end] == key;
    if (threadIdx.x == 0) stop = kThreads;
    __syncthreads();
    if (!goes_on) atomicMin(&stop, static_cast<int>(threadIdx.x));
    __syncthreads();
    const int at = stop;
    __syncthreads();
    if (at < kThreads) {
      last += at;
      break;
    }
  }
  auto load = [&](const float* row, int col) {
    if constexpr (VEC) return *reinterpret_cast<const float4*>(row + col);
    return make_float4(row[col], col + 1 < d ? row[col + 1] : 0.f, col + 2 < d ? row[col + 2] : 0.f, col + 3 < d ? row[col + 3] : 0.f);
  };
  auto add = [](float4& a, float4 b) { a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w; };
  __shared__ float4 parts[kThreads];
  const int group = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int col = blockIdx.y * kJoinSlice + lane * 4;
  const long long each = (last - w + 3) / 4, lo = w + 1 + group * each, hi = min(lo + each, last + 1);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (col < d) {
    if (group == 0) acc = load(tail + w * d, col);
#pragma unroll 8
    for (long long u = lo; u < hi; ++u) add(acc, load(head + u * d, col));
  }
  parts[threadIdx.x] = acc;
  __syncthreads();
  if (group == 0 && col < d) {
#pragma unroll
    for (int g = 1; g < 4; ++g) add(acc, parts[g * 64 + lane]);
    T* to = dw + key * static_cast<long long>(d) + col;
    put(to, acc.x * scale);
    if (VEC || col + 1 < d) put(to + 1, acc.y * scale);
    if (VEC || col + 2 < d) put(to + 2, acc.z * scale);
    if (VEC || col + 3 < d) put(to + 3, acc.w * scale);
  }
}

struct Plan {
  int window, slices, digit, passes;
  long long windows;
  size_t list, partials;                     // bytes of one list of n entries, of head or of tail
};

// Windows: short enough that about two CTAs an SM have one, between 8 and 64 tokens.  Longer ones leave fewer partial sums, and the
// longest run's are a chain: 16384 tokens of 4096 columns, a tenth of them one id, take 254 us in all with 32 and 246 with 64.
Plan plan_of(long long n, int d, long long v) {
  Plan p;
  p.slices = static_cast<int>(ceil_div(d, kSlice));
  const long long fit = n * p.slices / (2ll * sm_count());
  p.window = 8;
  while (p.window < 64 && p.window * 2 <= fit) p.window *= 2;
  p.windows = ceil_div(n, p.window);
  int bits = 1;
  while ((v >> bits) != 0) ++bits;           // keys are 0 to v
  p.passes = static_cast<int>(ceil_div(bits, kMaxDigit));
  p.digit = static_cast<int>(ceil_div(bits, p.passes));
  p.list = align_up(static_cast<size_t>(n) * 4, 256);
  p.partials = align_up(static_cast<size_t>(p.windows) * d * 4, 256);
  return p;
}

int check(const b200tp_embedding_args* a) {
  if (a == nullptr) return fail(B200TP_ERR_EMBEDDING_INPUT, "args is null");
  if (a->dtype != B200TP_F32 && a->dtype != B200TP_BF16) return fail(B200TP_ERR_EMBEDDING_INPUT, "tables must be fp32 or bf16");
  if (a->n < 0 || a->n > (1ll << 30)) return fail(B200TP_ERR_EMBEDDING_INPUT, "the number of tokens must lie in [0, 2^30]");
  if (a->d < 1 || a->d > (1 << 20)) return fail(B200TP_ERR_EMBEDDING_INPUT, "rows must have 1 to 2^20 columns");
  if (a->v < 1 || a->v >= (1ll << 31) - 1) return fail(B200TP_ERR_EMBEDDING_INPUT, "the table must have 1 to 2^31 - 2 rows");
  if (a->ids == nullptr && a->n > 0) return fail(B200TP_ERR_EMBEDDING_INPUT, "ids is null");
  if (a->row_stride < 0) return fail(B200TP_ERR_EMBEDDING_INPUT, "negative row stride");
  return B200TP_OK;
}

bool wide(const void* a, const void* b, long long stride, int d, int item) {
  return ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15) == 0 && stride * item % 16 == 0 && d % kCols == 0;
}

template <typename T, typename ID>
int launch_fwd(const b200tp_embedding_args* a, const void* weight, void* out, cudaStream_t stream, int* status) {
  const int parts = static_cast<int>(ceil_div(a->d, 1024));
  const long long blocks = ceil_div(a->n * parts, kThreads / 32);
  if (blocks > (1ll << 31) - 1) return fail(B200TP_ERR_EMBEDDING_INPUT, "too many tokens for one launch");
  auto go = [&](auto kernel) {
    return launch_pdl(kernel, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, stream, static_cast<const ID*>(a->ids),
                      static_cast<const T*>(weight), a->row_stride, a->n, a->d, parts, a->v, a->scale, static_cast<T*>(out), status);
  };
  B200TP_CUDA_OK(wide(weight, out, a->row_stride, a->d, sizeof(T)) ? go(embed_fwd_kernel<T, ID, true>) : go(embed_fwd_kernel<T, ID, false>));
  return B200TP_OK;
}

// Rows of a CTA of the direct kernel: about 64 kB, a multiple of eight.
int direct_rows(const b200tp_embedding_args* a) {
  const long long row = a->d * (a->dtype == B200TP_BF16 ? 2ll : 4ll);
  return static_cast<int>(std::max<long long>(8, kFillBytes / row / 8 * 8));
}
// Few tokens, and rows short enough that a CTA's eight are no long work.
bool direct(const b200tp_embedding_args* a) { return a->n <= kDirect && a->d <= 16384; }

template <typename T, typename ID>
int launch_direct(const b200tp_embedding_args* a, const void* dy, void* dw, cudaStream_t stream, int* status) {
  const int rows = direct_rows(a);
  auto go = [&](auto kernel) {
    return launch_pdl(kernel, dim3(static_cast<unsigned>(ceil_div(a->v, rows))), dim3(kDirectThreads), 0, stream,
                      static_cast<const ID*>(a->ids), static_cast<int>(a->n), a->v, a->padding_idx, rows, static_cast<const T*>(dy),
                      a->row_stride, a->d, a->scale, static_cast<T*>(dw), status);
  };
  B200TP_CUDA_OK(wide(dy, dw, a->row_stride, a->d, sizeof(T)) ? go(embed_direct_kernel<T, ID, true>) : go(embed_direct_kernel<T, ID, false>));
  return B200TP_OK;
}

constexpr size_t sort_smem(int digit) { return static_cast<size_t>(kSortWarps + 2) * (size_t{4} << digit); }

// The most shared memory a sort may ask for, once for each device.
int configure_sort() {
  static std::atomic<int> configured[64];
  int dev = 0;
  B200TP_CUDA_OK(cudaGetDevice(&dev));
  if (dev >= 0 && dev < 64 && configured[dev].load(std::memory_order_acquire)) return B200TP_OK;
  const int most = static_cast<int>(sort_smem(kMaxDigit));
  B200TP_CUDA_OK(cudaFuncSetAttribute(embed_sort_kernel<int>, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
  B200TP_CUDA_OK(cudaFuncSetAttribute(embed_sort_kernel<long long>, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
  if (dev >= 0 && dev < 64) configured[dev].store(1, std::memory_order_release);
  return B200TP_OK;
}

template <typename ID>
int launch_sort(const b200tp_embedding_args* a, const Sort& s, void* dw, cudaStream_t stream, int* status) {
  const long long bytes = a->v * a->d * (a->dtype == B200TP_BF16 ? 2 : 4);
  const int rc = configure_sort();
  if (rc) return rc;
  B200TP_CUDA_OK(launch_pdl(embed_sort_kernel<ID>, dim3(kCluster), dim3(kSortThreads), sort_smem(s.digit), stream, static_cast<const ID*>(a->ids), s,
                            status));
  B200TP_CUDA_OK(launch_pdl(embed_fill_kernel, dim3(static_cast<unsigned>(ceil_div(bytes, kFillBytes))), dim3(kSortThreads), 0, stream,
                            static_cast<uint4*>(dw), static_cast<long long>(bytes)));
  return B200TP_OK;
}

template <typename T>
int launch_sums(const b200tp_embedding_args* a, const Plan& p, const unsigned* keys, const unsigned* pos, const void* dy, void* dw,
                float* head, float* tail, cudaStream_t stream) {
  const bool vec = wide(dy, dw, a->row_stride, a->d, sizeof(T));
  const dim3 grid(static_cast<unsigned>(p.windows), p.slices);
  auto sum = [&](auto kernel) {
    return launch_pdl(kernel, grid, dim3(kThreads), 0, stream, keys, pos, a->n, p.window, a->v, static_cast<const T*>(dy), a->row_stride,
                      a->d, a->scale, static_cast<T*>(dw), head, tail);
  };
  B200TP_CUDA_OK(vec ? sum(embed_sum_kernel<T, true>) : sum(embed_sum_kernel<T, false>));
  if (p.windows == 1) return B200TP_OK;
  const dim3 join_grid(static_cast<unsigned>(p.windows), static_cast<unsigned>(ceil_div(a->d, kJoinSlice)));
  auto join = [&](auto kernel) {
    return launch_pdl(kernel, join_grid, dim3(kThreads), 0, stream, keys, a->n, p.window, a->v, a->d, a->scale, head, tail,
                      static_cast<T*>(dw));
  };
  B200TP_CUDA_OK(vec ? join(embed_join_kernel<T, true>) : join(embed_join_kernel<T, false>));
  return B200TP_OK;
}

}  // namespace
}  // namespace b200tp

using namespace b200tp;

extern "C" {

int b200tp_embedding_fwd(const b200tp_embedding_args* a, const void* weight, void* out, void* stream_v, int* status) {
  int rc = check(a);
  if (rc) return rc;
  if (a->n == 0) return B200TP_OK;
  if (weight == nullptr || out == nullptr) return fail(B200TP_ERR_EMBEDDING_INPUT, "weight / out is null");
  rc = require_sm100();
  if (rc) return rc;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  if (a->dtype == B200TP_BF16)
    return a->ids_int64 ? launch_fwd<__nv_bfloat16, long long>(a, weight, out, stream, status)
                        : launch_fwd<__nv_bfloat16, int>(a, weight, out, stream, status);
  return a->ids_int64 ? launch_fwd<float, long long>(a, weight, out, stream, status)
                      : launch_fwd<float, int>(a, weight, out, stream, status);
}

size_t b200tp_embedding_bwd_workspace_bytes(const b200tp_embedding_args* a) {
  if (check(a) != B200TP_OK || direct(a)) return 0;
  const Plan p = plan_of(a->n, a->d, a->v);
  return 4 * p.list + 2 * p.partials;
}

int b200tp_embedding_bwd(const b200tp_embedding_args* a, const void* d_out, void* d_weight, void* workspace,
                         size_t workspace_bytes, void* stream_v, int* status) {
  int rc = check(a);
  if (rc) return rc;
  if (d_weight == nullptr || (d_out == nullptr && a->n > 0)) return fail(B200TP_ERR_EMBEDDING_INPUT, "d_out / d_weight is null");
  if ((reinterpret_cast<uintptr_t>(d_weight) & 15) != 0) return fail(B200TP_ERR_EMBEDDING_INPUT, "d_weight must be 16-byte aligned");
  const size_t need = b200tp_embedding_bwd_workspace_bytes(a);
  if (need > 0 && (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 255) != 0 || workspace_bytes < need))
    return fail(B200TP_ERR_WORKSPACE, "embedding backward workspace missing, misaligned or smaller than " + std::to_string(need) + " bytes");
  rc = require_sm100();
  if (rc) return rc;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  if (direct(a)) {
    if (a->dtype == B200TP_BF16)
      return a->ids_int64 ? launch_direct<__nv_bfloat16, long long>(a, d_out, d_weight, stream, status)
                          : launch_direct<__nv_bfloat16, int>(a, d_out, d_weight, stream, status);
    return a->ids_int64 ? launch_direct<float, long long>(a, d_out, d_weight, stream, status)
                        : launch_direct<float, int>(a, d_out, d_weight, stream, status);
  }
  const Plan p = plan_of(a->n, a->d, a->v);
  char* ws = static_cast<char*>(workspace);
  Sort s;
  s.key_a = reinterpret_cast<unsigned*>(ws);
  s.pos_a = reinterpret_cast<unsigned*>(ws + p.list);
  s.key_b = reinterpret_cast<unsigned*>(ws + 2 * p.list);
  s.pos_b = reinterpret_cast<unsigned*>(ws + 3 * p.list);
  float* head = reinterpret_cast<float*>(ws + 4 * p.list);
  float* tail = reinterpret_cast<float*>(ws + 4 * p.list + p.partials);
  s.n = a->n;
  s.v = a->v;
  s.padding = a->padding_idx;
  s.digit = p.digit;
  s.passes = p.passes;
  rc = a->ids_int64 ? launch_sort<long long>(a, s, d_weight, stream, status) : launch_sort<int>(a, s, d_weight, stream, status);
  if (rc) return rc;
  const unsigned* keys = p.passes & 1 ? s.key_a : s.key_b;
  const unsigned* pos = p.passes & 1 ? s.pos_a : s.pos_b;
  return a->dtype == B200TP_BF16 ? launch_sums<__nv_bfloat16>(a, p, keys, pos, d_out, d_weight, head, tail, stream)
                                 : launch_sums<float>(a, p, keys, pos, d_out, d_weight, head, tail, stream);
}

}  // extern "C"
