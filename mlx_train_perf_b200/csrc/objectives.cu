// Objectives over per-token log-probabilities: the preference loss over pairs of sequences and the clipped policy loss
// with a KL term.  They stand behind the per-token losses of the vocabulary loss (core/loss.py:235-250 of the reference),
// where the reference's own training code has only the masked mean (adapters/mlx_lm.py:212-215).
//
// Tokens lie as (S, L) rows with a row stride, or as T packed tokens whose sequences are the ranges
// [cu[s], cu[s + 1]).  A token that its mask leaves out takes no part whatever it holds: values are selected, never
// multiplied by zero.
//
// Both losses are one pass over the tokens, then one block that joins the sequences' sums (up to eight blocks are one cluster, whose
// first block joins: no second launch), then (backward) one pass that writes the gradient.  A token costs 9 to 21 bytes and
// a few dozen operations, so long batches are bound by HBM and arithmetic, the usual ones by launches.  Nothing is zeroed
// beforehand (no counter, no atomics): sums are formed in a fixed order, and in double, since what is left after advantages
// of both signs cancel is small beside the terms.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "common.h"
#include "ptx.cuh"

namespace b200tp {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kJoinThreads = 1024;
constexpr unsigned kClusterMost = 8;
constexpr int kUnroll = 4;
constexpr int kShare = kThreads * 4;  // tokens of a block, on average
constexpr int kFewTokens = kThreads * 2;

struct Tokens {
  const void* cu;        // (S + 1) borders, or null: rows
  int cu_i64;
  long long seqs, length;            // length: of a row, or of all packed tokens
  int splits;                        // blocks a sequence
  long long x_stride, old_stride, ref_stride, mask_stride, adv_seq, adv_tok;
  const unsigned char* mask;
  float sign;                        // -1: the inputs are negative log-probabilities
};

struct PolicyRule {
  float log_low, log_high;           // log(1 - clip_low), log(1 + clip_high)
  float low, high;                   // 1 - clip_low, 1 + clip_high
  float kl_coef;                     // for the slopes; the loss takes it in double
  double kl_coef_loss;
  int kl_kind;
};

// What a block knows of one sequence's share of tokens.
struct alignas(32) Part {
  double loss, kl, count, clipped;
};

__device__ __forceinline__ float ld(const float* p) { return *p; }
__device__ __forceinline__ float ld(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void st(float* p, float v) { *p = v; }
__device__ __forceinline__ void st(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// Four adjacent values, aligned to their size; four mask bytes.
__device__ __forceinline__ void ld4(const float* p, float (&v)[4]) {
  const float4 a = *reinterpret_cast<const float4*>(p);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
}
__device__ __forceinline__ void ld4(const __nv_bfloat16* p, float (&v)[4]) {
  const uint2 a = *reinterpret_cast<const uint2*>(p);
  v[0] = __uint_as_float(a.x << 16);
  v[1] = __uint_as_float(a.x & 0xffff0000u);
  v[2] = __uint_as_float(a.y << 16);
  v[3] = __uint_as_float(a.y & 0xffff0000u);
}
__device__ __forceinline__ void st4(float* p, const float (&v)[4]) { *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void st4(__nv_bfloat16* p, const float (&v)[4]) {
  uint2 a;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&a);
  h[0] = __floats2bfloat162_rn(v[0], v[1]);
  h[1] = __floats2bfloat162_rn(v[2], v[3]);
  *reinterpret_cast<uint2*>(p) = a;
}
__device__ __forceinline__ void ld4(const unsigned char* p, bool (&v)[4]) {
  const uchar4 a = *reinterpret_cast<const uchar4*>(p);
  v[0] = a.x != 0; v[1] = a.y != 0; v[2] = a.z != 0; v[3] = a.w != 0;
}

// Which tokens of [lo, hi) are taken four at a time: those of [i0, i1), where every array's token i0 lies on a boundary of four.  The
// others, `rest` of them, one by one: single(v) for v in [0, rest).  Arrays that do not agree have no [i0, i1), and nor have shares of
// so few tokens that four a thread would leave threads idle (8 x 61 tokens: 8.7 us in all by fours, 7.4 one by one).
struct Fours {
  int lo, i0, i1, rest;
  __device__ __forceinline__ Fours(int lo_, int hi, int phase) : lo(lo_), i0(lo_), i1(lo_) {
    if (phase >= 0 && hi - lo > kFewTokens) {
      i0 = min(hi, lo + ((4 - ((phase + lo) & 3)) & 3));
      i1 = i0 + (hi - i0) / 4 * 4;
    }
    rest = (i0 - lo) + (hi - i1);
  }
  __device__ __forceinline__ int single(int v) const { return v < i0 - lo ? lo + v : i1 + v - (i0 - lo); }
};
// Where a row's first token lies in its four, as one number for arrays that agree, else -1.
template <typename T>
__device__ __forceinline__ int phase_of(const T* row) { return static_cast<int>(reinterpret_cast<uintptr_t>(row) / sizeof(T)) & 3; }
__device__ __forceinline__ int agree(int a, int b) { return a == b ? a : -1; }

__device__ __forceinline__ long long border(const Tokens& t, long long s) {
  const long long b = t.cu_i64 ? static_cast<const long long*>(t.cu)[s] : static_cast<const int*>(t.cu)[s];
  return min(max(b, 0ll), t.length);
}
// Tokens [lo, hi) of block (s, k); borders that do not rise give empty sequences, never an access outside.
__device__ __forceinline__ void share(const Tokens& t, long long s, int k, int& lo, int& hi) {
  lo = 0;
  hi = static_cast<int>(t.length);                                  // at most 2^30
  if (t.cu != nullptr) {
    lo = static_cast<int>(border(t, s));
    hi = max(static_cast<int>(border(t, s + 1)), lo);
  }
  const int per = (hi - lo + t.splits - 1) / t.splits;
  lo = static_cast<int>(min(lo + static_cast<long long>(per) * k, static_cast<long long>(hi)));
  hi = min(lo + per, hi);
}

// Sums of up to four values over a block of N threads, in a fixed order; all threads get them.
template <int N, int K>
__device__ __forceinline__ void block_sums(double (&v)[K], double (*shared)[K]) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  if ((threadIdx.x & 31) == 0)
#pragma unroll
    for (int k = 0; k < K; ++k) shared[threadIdx.x >> 5][k] = v[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    v[k] = (threadIdx.x & 31) < N / 32 ? shared[threadIdx.x & 31][k] : 0.;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  }
}

// exp(z) - 1 - z and exp(z) - 1 without cancellation: up to |z| = 1 the Taylor series to z^13 / 13!, whose first term left out
// is 2 z^12 / 14! < 3e-11 of the sum; beyond, the library's expm1.  (Log ratios of a few tenths then leave hardly a warp with both
// branches: a twelfth of the kernel's time against a series up to 1/2.)
__device__ __forceinline__ float exp_minus_line(float z, float* minus_one) {
  if (fabsf(z) > 1.f) {
    *minus_one = expm1f(z);
    return *minus_one - z;
  }
  float s = 1.f / 6227020800.f;
  s = fmaf(s, z, 1.f / 479001600.f);
  s = fmaf(s, z, 1.f / 39916800.f);
  s = fmaf(s, z, 1.f / 3628800.f);
  s = fmaf(s, z, 1.f / 362880.f);
  s = fmaf(s, z, 1.f / 40320.f);
  s = fmaf(s, z, 1.f / 5040.f);
  s = fmaf(s, z, 1.f / 720.f);
  s = fmaf(s, z, 1.f / 120.f);
  s = fmaf(s, z, 1.f / 24.f);
  s = fmaf(s, z, 1.f / 6.f);
  s = fmaf(s, z, 0.5f);
  s *= z * z;
  *minus_one = z + s;
  return s;
}

// A sequence's parts joined.  Up to eight: each thread of the warp does its own sequence `s`.  More: the warp's lanes share one.
__device__ __forceinline__ Part joined(const Part* parts, const Tokens& t, long long s) {
  Part p{0., 0., 0., 0.};
  for (int k = 0; k < t.splits; ++k) {
    const Part q = parts[s * t.splits + k];
    p.loss += q.loss;
    p.kl += q.kl;
    p.count += q.count;
    p.clipped += q.clipped;
  }
  return p;
}
__device__ __forceinline__ Part joined_by_warp(const Part* parts, const Tokens& t, long long s) {
  double v[4] = {0., 0., 0., 0.};
#pragma unroll 4
  for (int k = threadIdx.x & 31; k < t.splits; k += 32) {
    const Part q = parts[s * t.splits + k];
    v[0] += q.loss;
    v[1] += q.kl;
    v[2] += q.count;
    v[3] += q.clipped;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  return Part{v[0], v[1], v[2], v[3]};
}
constexpr int kFewParts = 8;

// One block of N threads: the sequences' sums, then the batch's.
struct PolicyJoin {
  int normalize;
  float *weights, *loss, *stats;
};
template <int N>
__device__ __forceinline__ void join(const Part* parts, const Tokens& t, const PolicyJoin& o) {
  const int normalize = o.normalize;
  float *weights = o.weights, *loss_out = o.loss, *stats = o.stats;
  __shared__ double sums[N / 32][4];
  double all[4] = {0., 0., 0., 0.};           // loss, kl, taken and clipped tokens
  const bool few = t.splits <= kFewParts;
  const int step = few ? N : N / 32;
  for (long long s = few ? threadIdx.x : threadIdx.x >> 5; s < t.seqs; s += step) {
    const Part p = few ? joined(parts, t, s) : joined_by_warp(parts, t, s);
    if (!few && (threadIdx.x & 31) != 0) continue;
    double l = p.loss;
    if (normalize == B200TP_NORMALIZE_SEQUENCE) {
      const double w = 1. / (static_cast<double>(t.seqs) * max(p.count, 1.));
      l *= w;
      weights[s] = static_cast<float>(w);
    }
    all[0] += l;
    all[1] += p.kl;
    all[2] += p.count;
    all[3] += p.clipped;
  }
  block_sums<N>(all, sums);
  const double loss = all[0], kl = all[1], count = all[2], clipped = all[3];
  if (threadIdx.x == 0) {
    const double per = 1. / max(count, 1.);
    if (normalize != B200TP_NORMALIZE_SEQUENCE) weights[0] = normalize == B200TP_NORMALIZE_TOKEN ? static_cast<float>(per) : 1.f;
    *loss_out = static_cast<float>(normalize == B200TP_NORMALIZE_TOKEN ? loss * per : loss);
    stats[0] = static_cast<float>(kl * per);
    stats[1] = static_cast<float>(clipped * per);
  }
}

// One block of N threads: pair i is the sequences i and P + i.  h = beta (l_i - l_{P + i}) - margin; out: the loss, the S rewards
// beta l_s, and for each sequence the weight that the loss's gradient gives every taken token of it.
struct PreferenceJoin {
  int kind;
  double beta, smoothing, margin;
  int average;
  float *loss, *rewards, *weights;
};
template <int N>
__device__ __forceinline__ void join(const Part* parts, const Tokens& t, const PreferenceJoin& o) {
  const int kind = o.kind, average = o.average;
  const double beta = o.beta, smoothing = o.smoothing, margin = o.margin;
  float *loss_out = o.loss, *rewards = o.rewards, *weights = o.weights;
  __shared__ double sums[N / 32][1];
  const long long pairs = t.seqs / 2;
  double total = 0.;
  const bool few = t.splits <= kFewParts;
  const int step = few ? N : N / 32;
  for (long long i = few ? threadIdx.x : threadIdx.x >> 5; i < pairs; i += step) {
    const Part c = few ? joined(parts, t, i) : joined_by_warp(parts, t, i);
    const Part r = few ? joined(parts, t, pairs + i) : joined_by_warp(parts, t, pairs + i);
    if (!few && (threadIdx.x & 31) != 0) continue;
    const double cs = average ? 1. / max(c.count, 1.) : 1., rs = average ? 1. / max(r.count, 1.) : 1.;
    const double lc = c.loss * cs, lr = r.loss * rs;
    const double h = beta * (lc - lr) - margin;
    double f, slope;
    if (kind == B200TP_PREFERENCE_SIGMOID) {
      const double e = exp(-fabs(h)), tail = log1p(e);
      f = (1. - smoothing) * (tail + max(-h, 0.));
      if (smoothing > 0.) f += smoothing * (tail + max(h, 0.));       // an infinite h must not meet a factor of zero
      slope = smoothing - (h >= 0. ? e : 1.) / (1. + e);             // smoothing - sigmoid(-h)
    } else if (kind == B200TP_PREFERENCE_HINGE) {
      f = h > 1. ? 0. : 1. - h;
      slope = h < 1. ? -1. : 0.;
    } else {
      const double off = (h - 0.5) / beta;
      f = off * off;
      slope = 2. * off / beta;
    }
    if (isnan(h)) f = slope = h;                                      // comparisons above would hide it
    total += f;
    const double w = t.sign * beta * slope / static_cast<double>(pairs);
    weights[i] = static_cast<float>(w * cs);
    weights[pairs + i] = static_cast<float>(-w * rs);
    rewards[i] = static_cast<float>(beta * lc);
    rewards[pairs + i] = static_cast<float>(beta * lr);
  }
  double all[1] = {total};
  block_sums<N>(all, sums);
  if (threadIdx.x == 0) *loss_out = static_cast<float>(all[0] / static_cast<double>(pairs));
}

template <typename Join>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const Part* parts, const Tokens t, const Join o) {
  griddep_wait();
  griddep_launch_dependents();
  join<kJoinThreads>(parts, t, o);
}

// The last step of a block of tokens that is one of a cluster: the first of them joins all parts.
template <typename Join>
__device__ __forceinline__ void join_in_cluster(const Part* parts, const Tokens& t, const Join& o) {
  cg::this_cluster().sync();                      // the parts of all blocks are written, and seen by all
  if (blockIdx.x == 0) join<kThreads>(parts, t, o);
}

// Per token:  u = x - o, ratio = exp(u);  clipped iff A > 0 and u > log(1 + high), or A < 0 and u < log(1 - low), which is
// where min(ratio A, clip(ratio) A) takes the constant (decided on u, an exact difference for near values, and not
// on the rounded exponential);  f = -A (clipped ? bound : ratio) + c kl;  slope = (clipped ? 0 : -A ratio) + c kl'.
// Slopes are kept without their weight (1 / count is known only after all tokens): 4 bytes written here and read
// again by the backward, where computing them anew would read 13 or more.
// Five blocks an SM (512 x 8192 tokens captured: 29.6 us; left alone 60 registers and 30.4 us, six blocks spill and take 29.9).
template <typename TX, typename TR, bool REF, bool CLUSTER>
__global__ void __launch_bounds__(kThreads, CLUSTER ? 1 : 5)
policy_tokens_kernel(const TX* __restrict__ x, const TR* __restrict__ old, const TR* __restrict__ ref,
                     const float* __restrict__ adv, const Tokens t, const PolicyRule r, float* __restrict__ slopes,
                     Part* __restrict__ parts, const PolicyJoin o) {
  griddep_wait();
  griddep_launch_dependents();
  __shared__ double sums[kThreads / 32][4];
  const long long s = blockIdx.x / t.splits;
  const int k = static_cast<int>(blockIdx.x % t.splits);
  const long long out_stride = t.cu != nullptr ? 0 : t.length;
  if (s >= t.seqs) {                 // packed tokens outside every sequence: no slope
    if (slopes != nullptr && s == t.seqs && k == 0 && t.cu != nullptr) {
      const long long first = border(t, 0), last = border(t, t.seqs);
      for (long long i = threadIdx.x; i < first; i += kThreads) slopes[i] = 0.f;
      for (long long i = max(first, last) + threadIdx.x; i < t.length; i += kThreads) slopes[i] = 0.f;
    }
    if constexpr (CLUSTER) join_in_cluster(parts, t, o);
    return;
  }
  int lo, hi;
  share(t, s, k, lo, hi);
  // rows, so that the loop indexes with 32 bits (126 instructions a token with 64, 100 with 32, 86 four tokens at a time)
  const TX* x_row = x + s * t.x_stride;
  const TR* old_row = old + s * t.old_stride;
  const TR* ref_row = REF ? ref + s * t.ref_stride : nullptr;
  const float* adv_row = adv + s * t.adv_seq;
  const unsigned char* mask_row = t.mask == nullptr ? nullptr : t.mask + s * t.mask_stride;
  float* slope_row = slopes == nullptr ? nullptr : slopes + s * out_stride;
  const bool adv_each = t.adv_tok != 0;
  const float adv_one = adv_each || lo >= hi ? 0.f : adv_row[0];
  double loss = 0., kl_sum = 0.;
  int count = 0, clips = 0;
  auto token = [&](bool on, float xv, float ov, float rv, float a) {          // the token's slope
    if (!on) return 0.f;
    const float u = t.sign * (xv - ov);
    const bool up = a > 0.f && u > r.log_high, down = a < 0.f && u < r.log_low, clipped = up || down;
    // without an advantage nothing, also where the ratio leaves fp32
    const float gain = a == 0.f && u < INFINITY ? 0.f : a * (clipped ? (up ? r.high : r.low) : expf(u));
    float slope = clipped ? 0.f : -gain;
    float kl = 0.f;
    if constexpr (REF) {
      const float z = t.sign * (rv - xv);
      float kl_slope;
      if (r.kl_kind == B200TP_KL_K3) {
        kl = exp_minus_line(z, &kl_slope);
        kl_slope = -kl_slope;
      } else if (r.kl_kind == B200TP_KL_K2) {
        kl = 0.5f * z * z;
        kl_slope = -z;
      } else {
        kl = -z;
        kl_slope = 1.f;
      }
      if (r.kl_coef != 0.f) slope = fmaf(r.kl_coef, kl_slope, slope);
      kl_sum += kl;
    }
    loss -= gain;
    count += 1;
    clips += clipped;
    return t.sign * slope;
  };
  int phase = agree(phase_of(x_row), phase_of(old_row));
  if constexpr (REF) phase = agree(phase, phase_of(ref_row));
  if (adv_each) phase = t.adv_tok == 1 ? agree(phase, phase_of(adv_row)) : -1;
  if (mask_row != nullptr) phase = agree(phase, phase_of(mask_row));
  if (slope_row != nullptr) phase = agree(phase, phase_of(slope_row));
  const Fours f(lo, hi, phase);
  for (int i = f.i0 + 4 * threadIdx.x; i < f.i1; i += 4 * kThreads) {
    float xv[4], ov[4], rv[4] = {}, av[4] = {adv_one, adv_one, adv_one, adv_one}, sv[4];
    bool on[4] = {true, true, true, true};
    ld4(x_row + i, xv);
    ld4(old_row + i, ov);
    if constexpr (REF) ld4(ref_row + i, rv);
    if (adv_each) ld4(adv_row + i, av);
    if (mask_row != nullptr) ld4(mask_row + i, on);
#pragma unroll
    for (int j = 0; j < 4; ++j) sv[j] = token(on[j], xv[j], ov[j], rv[j], av[j]);
    if (slope_row != nullptr) st4(slope_row + i, sv);
  }
  for (int base = threadIdx.x; base < f.rest; base += kThreads * kUnroll) {
    float xv[kUnroll], ov[kUnroll], rv[kUnroll] = {}, av[kUnroll];
    bool on[kUnroll];
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {                               // all loads first
      const int i = f.single(min(base + j * kThreads, f.rest - 1));
      on[j] = mask_row == nullptr || mask_row[i] != 0;
      xv[j] = ld(x_row + i);
      ov[j] = ld(old_row + i);
      if constexpr (REF) rv[j] = ld(ref_row + i);
      av[j] = adv_each ? adv_row[i * t.adv_tok] : adv_one;
    }
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      if (base + j * kThreads >= f.rest) break;
      const float slope = token(on[j], xv[j], ov[j], rv[j], av[j]);
      if (slope_row != nullptr) slope_row[f.single(base + j * kThreads)] = slope;
    }
  }
  double all[4] = {loss, kl_sum, static_cast<double>(count), static_cast<double>(clips)};       // counts are exact
  block_sums<kThreads>(all, sums);
  if (threadIdx.x == 0) {
    // The KL term joins the loss in double: gains of both signs cancel, and rounded together with one of them it would carry its error.
    // An infinite KL that is only reported stays out.
    if (r.kl_coef_loss != 0.) all[0] += r.kl_coef_loss * all[1];
    parts[blockIdx.x] = Part{all[0], all[1], all[2], all[3]};
  }
  if constexpr (CLUSTER) join_in_cluster(parts, t, o);
}

// Sum of the masked log ratios x - r of a sequence's share.
template <typename TX, typename TR, bool REF, bool CLUSTER>
__global__ void __launch_bounds__(kThreads)
preference_tokens_kernel(const TX* __restrict__ x, const TR* __restrict__ ref, const Tokens t, Part* __restrict__ parts,
                         const PreferenceJoin o) {
  griddep_wait();
  griddep_launch_dependents();
  __shared__ double sums[kThreads / 32][2];
  const long long s = blockIdx.x / t.splits;
  if constexpr (CLUSTER) {
    if (s >= t.seqs) {                // fills up the cluster
      join_in_cluster(parts, t, o);
      return;
    }
  }
  int lo, hi;
  share(t, s, static_cast<int>(blockIdx.x % t.splits), lo, hi);
  const TX* x_row = x + s * t.x_stride;
  const TR* ref_row = REF ? ref + s * t.ref_stride : nullptr;
  const unsigned char* mask_row = t.mask == nullptr ? nullptr : t.mask + s * t.mask_stride;
  double sum = 0.;
  int count = 0;
  auto token = [&](bool on, float xv, float rv) {
    if (!on) return;
    sum += REF ? static_cast<double>(xv) - rv : xv;
    count += 1;
  };
  int phase = phase_of(x_row);
  if constexpr (REF) phase = agree(phase, phase_of(ref_row));
  if (mask_row != nullptr) phase = agree(phase, phase_of(mask_row));
  const Fours f(lo, hi, phase);
#pragma unroll 2
  for (int i = f.i0 + 4 * threadIdx.x; i < f.i1; i += 4 * kThreads) {
    float xv[4], rv[4] = {};
    bool on[4] = {true, true, true, true};
    ld4(x_row + i, xv);
    if constexpr (REF) ld4(ref_row + i, rv);
    if (mask_row != nullptr) ld4(mask_row + i, on);
#pragma unroll
    for (int j = 0; j < 4; ++j) token(on[j], xv[j], rv[j]);
  }
  for (int base = threadIdx.x; base < f.rest; base += kThreads * kUnroll) {
    float xv[kUnroll], rv[kUnroll] = {};
    bool on[kUnroll];
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      const int i = f.single(min(base + j * kThreads, f.rest - 1));
      on[j] = base + j * kThreads < f.rest && (mask_row == nullptr || mask_row[i] != 0);
      xv[j] = ld(x_row + i);
      if constexpr (REF) rv[j] = ld(ref_row + i);
    }
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) token(on[j], xv[j], rv[j]);
  }
  double all[2] = {sum * t.sign, static_cast<double>(count)};
  block_sums<kThreads>(all, sums);
  if (threadIdx.x == 0) parts[blockIdx.x] = Part{all[0], 0., all[1], 0.};
  if constexpr (CLUSTER) join_in_cluster(parts, t, o);
}

// grad = upstream * weight * (slopes ? slope : mask).  `per_seq`: a weight for each sequence, else one.
template <typename TX, bool SLOPES>
__global__ void __launch_bounds__(kThreads)
objective_grad_kernel(const float* __restrict__ slopes, const float* __restrict__ weights, int per_seq,
                      const float* __restrict__ upstream, const Tokens t, TX* __restrict__ grad) {
  griddep_wait();
  griddep_launch_dependents();
  const long long s = blockIdx.x / t.splits;
  const int k = static_cast<int>(blockIdx.x % t.splits);
  const long long out_stride = t.cu != nullptr ? 0 : t.length;
  if (s == t.seqs) {
    if (k == 0 && t.cu != nullptr) {
      const long long first = border(t, 0), last = border(t, t.seqs);
      for (long long i = threadIdx.x; i < first; i += kThreads) st(grad + i, 0.f);
      for (long long i = max(first, last) + threadIdx.x; i < t.length; i += kThreads) st(grad + i, 0.f);
    }
    return;
  }
  int lo, hi;
  share(t, s, k, lo, hi);
  const unsigned char* mask_row = t.mask == nullptr ? nullptr : t.mask + s * t.mask_stride;
  const float* slope_row = SLOPES ? slopes + s * out_stride : nullptr;
  TX* grad_row = grad + s * out_stride;
  const float w = *upstream * weights[per_seq ? s : 0];
  int phase = phase_of(grad_row);
  if (mask_row != nullptr) phase = agree(phase, phase_of(mask_row));
  if constexpr (SLOPES) phase = agree(phase, phase_of(slope_row));
  const Fours f(lo, hi, phase);
#pragma unroll 2
  for (int i = f.i0 + 4 * threadIdx.x; i < f.i1; i += 4 * kThreads) {
    float v[4] = {1.f, 1.f, 1.f, 1.f};
    bool on[4] = {true, true, true, true};
    if constexpr (SLOPES) ld4(slope_row + i, v);
    if (mask_row != nullptr) ld4(mask_row + i, on);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = on[j] ? w * v[j] : 0.f;
    st4(grad_row + i, v);
  }
#pragma unroll 4
  for (int v = threadIdx.x; v < f.rest; v += kThreads) {
    const int i = f.single(v);
    st(grad_row + i, mask_row == nullptr || mask_row[i] != 0 ? w * (SLOPES ? slope_row[i] : 1.f) : 0.f);
  }
}

// Blocks a sequence: about 1024 tokens each on average, at most eight blocks an SM in all and at most 512 a sequence.
int splits_of(long long seqs, long long length, bool packed) {
  const int64_t mean = packed ? ceil_div(length, seqs) : length;
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>(512, 8ll * sm_count() / seqs));
  return static_cast<int>(std::max<int64_t>(1, std::min(most, ceil_div(mean, kShare))));
}

int check(const b200tp_objective_args* a) {
  if (a == nullptr) return fail(B200TP_ERR_LOSS_INPUT, "args is null");
  if (a->seqs < 1 || a->seqs > (1ll << 26)) return fail(B200TP_ERR_LOSS_INPUT, "the number of sequences must lie in [1, 2^26]");
  if (a->length < 0) return fail(B200TP_ERR_LOSS_INPUT, "negative length");
  if (a->length > (1ll << 30)) return fail(B200TP_ERR_LOSS_INPUT, "a row (or the packed batch) holds at most 2^30 tokens");
  if ((a->dtype != B200TP_F32 && a->dtype != B200TP_BF16) || (a->other_dtype != B200TP_F32 && a->other_dtype != B200TP_BF16))
    return fail(B200TP_ERR_LOSS_INPUT, "log-probabilities must be fp32 or bf16");
  if (a->logps == nullptr && a->length > 0) return fail(B200TP_ERR_LOSS_INPUT, "logps is null");
  return B200TP_OK;
}

Tokens tokens(const b200tp_objective_args* a) {
  Tokens t;
  t.cu = a->cu_seqlens;
  t.cu_i64 = a->cu_is_int64;
  t.seqs = a->seqs;
  t.length = a->length;
  t.splits = splits_of(a->seqs, a->length, a->cu_seqlens != nullptr);
  t.x_stride = a->logps_stride;
  t.old_stride = a->old_stride;
  t.ref_stride = a->ref_stride;
  t.mask_stride = a->mask_stride;
  t.adv_seq = a->advantage_stride_seq;
  t.adv_tok = a->advantage_stride_token;
  t.mask = static_cast<const unsigned char*>(a->mask);
  t.sign = a->from_nll ? -1.f : 1.f;
  return t;
}

unsigned blocks_of(const Tokens& t, bool outside) {
  return static_cast<unsigned>(t.seqs * t.splits + (outside && t.cu != nullptr ? 1 : 0));
}

int check_workspace(const b200tp_objective_args* a, void* workspace, size_t bytes) {
  const size_t need = b200tp_objective_workspace_bytes(a);
  if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 255) != 0 || bytes < need)
    return fail(B200TP_ERR_WORKSPACE, "objective workspace missing, misaligned or smaller than " + std::to_string(need) + " bytes");
  return B200TP_OK;
}

// A tokens kernel and its join: one launch of a cluster of 1, 2, 4 or 8 blocks where that holds them all (8 x 61 tokens, forward and
// backward: 6.5 us on the device against 7.8, and 2 us less of host time), else two launches.
template <typename Join, typename Go>
int launch_both(unsigned blocks, const Part* parts, const Tokens& t, const Join& o, cudaStream_t stream, Go go) {
  if (blocks <= kClusterMost) {
    unsigned size = 1;
    while (size < blocks) size *= 2;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = size;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(size);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    B200TP_CUDA_OK(go(cfg, std::true_type{}));
    return B200TP_OK;
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 1 : 0;
  B200TP_CUDA_OK(go(cfg, std::false_type{}));
  B200TP_CUDA_OK(launch_pdl(join_kernel<Join>, dim3(1), dim3(kJoinThreads), 0, stream, parts, t, o));
  return B200TP_OK;
}

template <typename TX, typename TR>
int launch_policy(const b200tp_objective_args* a, const Tokens& t, const PolicyRule& r, float* slopes, Part* parts,
                  const PolicyJoin& o, cudaStream_t stream) {
  const TX* x = static_cast<const TX*>(a->logps);
  const TR *old = static_cast<const TR*>(a->old_logps), *ref = static_cast<const TR*>(a->ref_logps);
  const float* adv = static_cast<const float*>(a->advantages);
  return launch_both(blocks_of(t, slopes != nullptr), parts, t, o, stream, [&](const cudaLaunchConfig_t& cfg, auto cluster) {
    constexpr bool kIn = decltype(cluster)::value;
    return ref != nullptr ? cudaLaunchKernelEx(&cfg, policy_tokens_kernel<TX, TR, true, kIn>, x, old, ref, adv, t, r, slopes, parts, o)
                          : cudaLaunchKernelEx(&cfg, policy_tokens_kernel<TX, TR, false, kIn>, x, old, ref, adv, t, r, slopes, parts, o);
  });
}

template <typename TX, typename TR>
int launch_preference(const b200tp_objective_args* a, const Tokens& t, Part* parts, const PreferenceJoin& o, cudaStream_t stream) {
  const TX* x = static_cast<const TX*>(a->logps);
  const TR* ref = static_cast<const TR*>(a->ref_logps);
  return launch_both(blocks_of(t, false), parts, t, o, stream, [&](const cudaLaunchConfig_t& cfg, auto cluster) {
    constexpr bool kIn = decltype(cluster)::value;
    return ref != nullptr ? cudaLaunchKernelEx(&cfg, preference_tokens_kernel<TX, TR, true, kIn>, x, ref, t, parts, o)
                          : cudaLaunchKernelEx(&cfg, preference_tokens_kernel<TX, TR, false, kIn>, x, ref, t, parts, o);
  });
}

}  // namespace
}  // namespace b200tp

using namespace b200tp;

extern "C" {

size_t b200tp_objective_workspace_bytes(const b200tp_objective_args* a) {
  if (check(a) != B200TP_OK) return 0;
  return align_up(static_cast<size_t>(a->seqs) * splits_of(a->seqs, a->length, a->cu_seqlens != nullptr) * sizeof(Part), 256);
}

int b200tp_preference_loss_fwd(const b200tp_objective_args* a, int32_t kind, double beta, double label_smoothing,
                               double margin, int32_t average, float* loss, float* rewards, float* weights,
                               void* workspace, size_t workspace_bytes, void* stream_v) {
  int rc = check(a);
  if (rc) return rc;
  if (a->seqs % 2 != 0) return fail(B200TP_ERR_LOSS_INPUT, "a preference loss needs an even number of sequences");
  if (kind != B200TP_PREFERENCE_SIGMOID && kind != B200TP_PREFERENCE_HINGE && kind != B200TP_PREFERENCE_SQUARED)
    return fail(B200TP_ERR_LOSS_INPUT, "unknown kind of preference loss");
  if (!(beta > 0.)) return fail(B200TP_ERR_LOSS_INPUT, "beta must be positive");
  if (loss == nullptr || rewards == nullptr || weights == nullptr) return fail(B200TP_ERR_LOSS_INPUT, "null output");
  rc = check_workspace(a, workspace, workspace_bytes);
  if (rc) return rc;
  rc = require_sm100();
  if (rc) return rc;
  const Tokens t = tokens(a);
  Part* parts = static_cast<Part*>(workspace);
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  const PreferenceJoin o{kind, beta, label_smoothing, margin, average, loss, rewards, weights};
  if (a->dtype == B200TP_BF16)
    return a->other_dtype == B200TP_BF16 ? launch_preference<__nv_bfloat16, __nv_bfloat16>(a, t, parts, o, stream)
                                         : launch_preference<__nv_bfloat16, float>(a, t, parts, o, stream);
  return a->other_dtype == B200TP_BF16 ? launch_preference<float, __nv_bfloat16>(a, t, parts, o, stream)
                                       : launch_preference<float, float>(a, t, parts, o, stream);
}

int b200tp_policy_loss_fwd(const b200tp_objective_args* a, double clip_low, double clip_high, double kl_coef, int32_t kl_kind,
                           int32_t normalize, float* loss, float* stats, float* slopes, float* weights, void* workspace,
                           size_t workspace_bytes, void* stream_v) {
  int rc = check(a);
  if (rc) return rc;
  if (!(clip_low >= 0. && clip_low <= 1.) || !(clip_high >= 0.))
    return fail(B200TP_ERR_LOSS_INPUT, "clip_low must lie in [0, 1] and clip_high must not be negative");
  if (kl_kind < B200TP_KL_K1 || kl_kind > B200TP_KL_K3) return fail(B200TP_ERR_LOSS_INPUT, "unknown kind of KL term");
  if (normalize < B200TP_NORMALIZE_TOKEN || normalize > B200TP_NORMALIZE_SUM)
    return fail(B200TP_ERR_LOSS_INPUT, "unknown normalisation");
  if (kl_coef != 0. && a->ref_logps == nullptr && a->length > 0) return fail(B200TP_ERR_LOSS_INPUT, "a KL term needs ref_logps");
  if (loss == nullptr || stats == nullptr || weights == nullptr) return fail(B200TP_ERR_LOSS_INPUT, "null output");
  if (a->length > 0 && (a->old_logps == nullptr || a->advantages == nullptr))
    return fail(B200TP_ERR_LOSS_INPUT, "old_logps / advantages is null");
  rc = check_workspace(a, workspace, workspace_bytes);
  if (rc) return rc;
  rc = require_sm100();
  if (rc) return rc;
  const Tokens t = tokens(a);
  PolicyRule r;
  r.log_low = static_cast<float>(std::log1p(-clip_low));      // clip_low = 1: minus infinity, nothing lies below
  r.log_high = static_cast<float>(std::log1p(clip_high));
  r.low = static_cast<float>(1. - clip_low);
  r.high = static_cast<float>(1. + clip_high);
  r.kl_coef = static_cast<float>(kl_coef);
  r.kl_coef_loss = kl_coef;
  r.kl_kind = kl_kind;
  Part* parts = static_cast<Part*>(workspace);
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  const PolicyJoin o{normalize, weights, loss, stats};
  if (a->dtype == B200TP_BF16)
    return a->other_dtype == B200TP_BF16 ? launch_policy<__nv_bfloat16, __nv_bfloat16>(a, t, r, slopes, parts, o, stream)
                                         : launch_policy<__nv_bfloat16, float>(a, t, r, slopes, parts, o, stream);
  return a->other_dtype == B200TP_BF16 ? launch_policy<float, __nv_bfloat16>(a, t, r, slopes, parts, o, stream)
                                       : launch_policy<float, float>(a, t, r, slopes, parts, o, stream);
}

int b200tp_objective_bwd(const b200tp_objective_args* a, const float* slopes, const float* weights, int32_t per_sequence,
                         const float* upstream, void* grad, void* stream_v) {
  int rc = check(a);
  if (rc) return rc;
  if (weights == nullptr || upstream == nullptr || (grad == nullptr && a->length > 0))
    return fail(B200TP_ERR_LOSS_INPUT, "weights / upstream / grad is null");
  rc = require_sm100();
  if (rc) return rc;
  const Tokens t = tokens(a);
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  auto go = [&](auto kernel, auto* out) {
    return launch_pdl(kernel, dim3(blocks_of(t, true)), dim3(kThreads), 0, stream, slopes, weights, per_sequence, upstream, t, out);
  };
  if (a->dtype == B200TP_BF16) {
    auto* out = static_cast<__nv_bfloat16*>(grad);
    B200TP_CUDA_OK(slopes != nullptr ? go(objective_grad_kernel<__nv_bfloat16, true>, out)
                                     : go(objective_grad_kernel<__nv_bfloat16, false>, out));
  } else {
    auto* out = static_cast<float*>(grad);
    B200TP_CUDA_OK(slopes != nullptr ? go(objective_grad_kernel<float, true>, out) : go(objective_grad_kernel<float, false>, out));
  }
  return B200TP_OK;
}

}  // extern "C"
