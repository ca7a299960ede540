// One AdamW step over many tensors, moments in 32 or in 8 bits, with or without fp32 masters of bf16 parameters: what the
// reference leaves to mlx.optimizers.AdamW (its train steps; plan/estimate.py:57-135 books the two moments).
//
// Everything is read once and written once: 28 bytes an element for bf16 parameters with fp32 masters and fp32 moments, 10 for
// bf16 parameters with 8-bit moments.  HBM bounds the first.  The second leaves time for about 56 instructions an element at
// HBM's rate, and written plainly (a rounded square root and quotient, selections for values that are not finite) it takes 79; so its
// arithmetic works on pairs of fp32 values (fma.rn.f32x2), takes roots and quotients from approximate ones with one corrected step,
// and tests a thread's eight elements together for what is rare.
//
// The table of tensors travels in the launch's own parameters: no copy to the device, no workspace, nothing that two captured
// graphs would share.  A CTA takes some thousands of elements of one tensor; a warp takes blocks of 256, the elements that share a scale.
//
// 8-bit moments.  v: e4m3 codes of sqrt(v), scale rmax / 448 of the block, rounded up or down by a dither that is fixed by position and
// step: beta2 moves v by a thousandth a step, far less than half the distance of two codes, and rounding to nearest would hold
// every v where it is.  A v that is not zero is never coded as zero: the update divides by it.  An element one of whose moments is
// not finite gets NaN for both (and so does its parameter); the block's scales are taken from the others.
//
// m: e4m3 codes, scale amax / 448, to nearest where that cannot hold a code that no gradient feeds, else by a dither of its own.  A held
// m is worse than a held v: v goes on falling, m / sqrt(v) grows, and the parameter drifts without a gradient.  Times 0.9 a code of
// mantissa 8 to 15 falls by 0.8 to 1.5 of a distance (half as wide below 8) and is never rounded back; up to beta1 = 0.9 these go to
// nearest.  Below 2^-6 the distance stays 2^-9, and code 4 comes back from 3.6: codes there are dithered wherever the gradient
// adds less than 2^-6 too.  Above beta1 = 0.9 every m is dithered (at 0.95 code 9 comes back from 8.55).  A warp that meets an old
// code below 2^-6 takes a form of the step that looks; all others ask once for eight elements.  789 M elements: 1263 us at full
// clocks; sustained at the power cap 1475 us (1435 with every m to nearest), 1935 us with all dithered.
//
// Moments, roots, scales and codes are, bit for bit, those of the definition computed in fp32 with each operation rounded by itself:
// codes depend on the last bit of what is rounded, so anything else gives other codes here and there (sums fused with
// their products: 64 codes of m in 56 M; scales folded into the factors besides would be 4 % faster).
//
// Moments of 1e-30 and less, and roots of 4e-19 and less, are held as zero: the factor to their codes would overflow.
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <iterator>
#include <type_traits>
#include <vector>

#include "common.h"
#include "ptx.cuh"

namespace b200tp {
namespace {

constexpr int kThreads = 256;
constexpr int kBlock = 256;                 // elements that share a scale; tensors start at multiples of it in the states
constexpr int kRound = 4096;                // elements that a CTA loads at once: two blocks a warp
// Elements of one CTA.  8-bit moments: one round (two in a loop need 120 registers or spill: a quarter and a seventh slower at 789 M
// elements).  32 bits: two, which halves the searches of the table (unaligned tensors: 100 % of the copy rate against 92 %).
template <int BITS>
constexpr int kChunk = BITS == 8 ? kRound : 2 * kRound;
constexpr int kTensors = 600;               // of one launch: 26 kB of its parameters
constexpr int kNear = 64;                   // entries of the coarse index
constexpr int kFew = 48;                    // of the small form: 2 kB, 5.9 us of host time for 48 tensors against 11.3 (one: 4.5, 6.3)

struct Rule {
  float beta1, beta2, one_beta1, one_beta2;
  float eps, decay;                         // decay: 1 - lr weight_decay
  float rate;                               // lr / (1 - beta1^t)
  float root;                               // 1 / sqrt(1 - beta2^t)
  float grad_scale;
  const float* grad_scale_ptr;              // or null
  unsigned step;
  int dither_m;                             // every m, not only the small ones that nothing feeds
};

struct States {
  const void* m;
  const void* v;
  const float2* scales;
  const float* master;
  void* m_out;
  void* v_out;
  float2* scales_out;
  float* master_out;
};

template <int N>
struct Table {
  const void* p[N];
  const void* g[N];
  void* out[N];
  long long numel[N];
  long long at[N];                          // of the tensor's first element in the states
  int first[N + 1];                         // chunk of the tensor's first element
  short near[kNear + 1];                    // the tensor of chunk k << shift, the last one behind the end
  int shift;
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vec, int n, float (&v)[8]) {
  if (vec && n >= 8) {
    if constexpr (sizeof(T) == 2) {
      const uint4 u = __ldcs(reinterpret_cast<const uint4*>(p));
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    } else {
      const float4 a = __ldcs(reinterpret_cast<const float4*>(p)), b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (sizeof(T) == 2) v[i] = i < n ? __bfloat162float(p[i]) : 0.f;
      else v[i] = i < n ? p[i] : 0.f;
    }
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, bool vec, int n, const float (&v)[8]) {
  if (vec && n >= 8) {
    if constexpr (sizeof(T) == 2) {
      uint4 u;
      __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      __stcs(reinterpret_cast<uint4*>(p), u);
    } else {
      __stcs(reinterpret_cast<float4*>(p), make_float4(v[0], v[1], v[2], v[3]));
      __stcs(reinterpret_cast<float4*>(p) + 1, make_float4(v[4], v[5], v[6], v[7]));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) {
        if constexpr (sizeof(T) == 2) p[i] = __float2bfloat16_rn(v[i]);
        else p[i] = v[i];
      }
  }
}

// Pairs of fp32 values, one instruction for two.
struct alignas(8) Pair {
  float x, y;
};
__device__ __forceinline__ unsigned long long bits_of(Pair a) {
  unsigned long long u;
  asm("mov.b64 %0, {%1, %2};" : "=l"(u) : "f"(a.x), "f"(a.y));
  return u;
}
__device__ __forceinline__ Pair pair_of(unsigned long long u) {
  Pair a;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a.x), "=f"(a.y) : "l"(u));
  return a;
}
__device__ __forceinline__ Pair both(float v) { return Pair{v, v}; }
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  unsigned long long d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(bits_of(a)), "l"(bits_of(b)), "l"(bits_of(c)));
  return pair_of(d);
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  unsigned long long d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits_of(a)), "l"(bits_of(b)));
  return pair_of(d);
}
// Two scalar additions: a packed one is fused with the product before it, which then goes unrounded.
__device__ __forceinline__ Pair add2(Pair a, Pair b) { return Pair{__fadd_rn(a.x, b.x), __fadd_rn(a.y, b.y)}; }
__device__ __forceinline__ float rsqrt_ftz(float v) {
  float q;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(q) : "f"(v));
  return q;
}
__device__ __forceinline__ float rcp_ftz(float v) {
  float q;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q) : "f"(v));
  return q;
}

// a / b rounded once, from an approximate reciprocal of b: the product corrected by its exact remainder.
__device__ __forceinline__ Pair divide2(Pair a, Pair minus_b, Pair over_b) {
  const Pair q = mul2(a, over_b);
  return fma2(fma2(q, minus_b, a), over_b, q);
}
constexpr float kNoRoot = 4e-19f;           // roots up to here stand for zero: the root of 1e-37 is 3.2e-19

// Two e4m3 codes of a word, the lower or the upper ones.
__device__ __forceinline__ Pair decode2(uint32_t w, int upper) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(upper ? w >> 16 : w & 0xffffu), __NV_E4M3);
  const float2 f = __half22float2(__half2(h));
  return Pair{f.x, f.y};
}

// 32 mixed bits of a pair of positions and the step: xor-shifts by 16, 15, 16 and multipliers between them, which are those of
// C. Wellons's published search for 32-bit integer hashes of low bias (2018), the last one's top bit cleared.
__device__ __forceinline__ uint32_t mix(uint32_t pair, uint32_t step) {
  uint32_t x = (pair + step * 0x3504F333u) * 0x1E3779B1u;
  x = (x ^ (x >> 16)) * 0x7FEB352Du;
  x = (x ^ (x >> 15)) * 0x046CA68Bu;
  return x ^ (x >> 16);
}

// y >= 0 to the e4m3 value below or above, up with a probability of the distance (dither uniform in [0, 2^20)).  Below 2^-6, where e4m3
// values lie 2^-9 apart, 2^-6 is added first: sums in [2^-6, 2^-5) lie as far apart.
__device__ __forceinline__ float dithered(float y, uint32_t dither) {
  const float lift = y < 0x1p-6f ? 0x1p-6f : 0.f;
  const uint32_t u = __float_as_uint(y + lift) + dither;
  return __uint_as_float(u & 0xfff00000u) - lift;
}

// Eight elements as they lie in memory.
template <typename T>
struct Raw8 {
  uint4 w[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ void fetch8(const T* p, bool vec, int n, Raw8<T>& r) {
  if (vec && n >= 8) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) r.w[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
  } else {
    T v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : T(0.f);
    memcpy(&r, v, sizeof(v));
  }
}
__device__ __forceinline__ void unpack(const Raw8<__nv_bfloat16>& r, Pair (&v)[4]) {
  const uint32_t w[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = Pair{__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u)};
}
__device__ __forceinline__ void unpack(const Raw8<float>& r, Pair (&v)[4]) {
  v[0] = Pair{__uint_as_float(r.w[0].x), __uint_as_float(r.w[0].y)};
  v[1] = Pair{__uint_as_float(r.w[0].z), __uint_as_float(r.w[0].w)};
  v[2] = Pair{__uint_as_float(r.w[1].x), __uint_as_float(r.w[1].y)};
  v[3] = Pair{__uint_as_float(r.w[1].z), __uint_as_float(r.w[1].w)};
}

// 8-bit moments of eight elements: (codes, scales) and gradients in, parameters moved, (codes, scales) out.
// m = beta1 (sm code) + one_beta1 g;  v = beta2 (sr code)^2 + (one_beta2 g) g, g times grad_scale before;  sqrt(v) from v rsqrt(v) and
// one Newton step with the exact remainder.  1e-37 is added to the old v, which keeps rsqrt finite and changes no v above 1e-30; what is
// then below 1.6e-37 is zero.  `pair`: half the first element's place in the states, which fixes the dither.  LOOK: m that is not to
// go to nearest is dithered, with the bits of the complement of `pair`.
template <bool LOOK>
__device__ __forceinline__ void step8(uint2& mc, uint2& vc, float2& sc, const Pair (&g)[4], Pair (&p)[4], const Rule& r,
                                      uint32_t pair) {
  Pair m[4], root[4];
  const Pair old_m = both(sc.x), old_r = both(sc.y);
  float ma = 0.f;
  uint32_t top = 0, by_dither = 0;                                  // by_dither: bit k for element k
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const Pair cm = decode2(i < 2 ? mc.x : mc.y, i & 1), cv = decode2(i < 2 ? vc.x : vc.y, i & 1);
    const Pair fed = mul2(g[i], both(r.one_beta1));
    m[i] = add2(mul2(mul2(cm, old_m), both(r.beta1)), fed);
    if constexpr (LOOK) {
      if (r.dither_m || (fabsf(cm.x) < 0x1p-6f && fabsf(fed.x) < 0x1p-6f * sc.x)) by_dither |= 1u << (2 * i);
      if (r.dither_m || (fabsf(cm.y) < 0x1p-6f && fabsf(fed.y) < 0x1p-6f * sc.x)) by_dither |= 2u << (2 * i);
    }
    const Pair old_root = mul2(cv, old_r);
    const Pair v = add2(fma2(mul2(old_root, old_root), both(r.beta2), both(1e-37f)), mul2(mul2(g[i], both(r.one_beta2)), g[i]));
    const Pair q = Pair{rsqrt_ftz(v.x), rsqrt_ftz(v.y)};
    const Pair t = mul2(v, q);
    root[i] = fma2(Pair{fmaf(-t.x, t.x, v.x), fmaf(-t.y, t.y, v.y)}, mul2(q, both(0.5f)), t);
    const Pair d = fma2(root[i], both(r.root), both(r.eps));
    const Pair move = mul2(m[i], Pair{rcp_ftz(d.x), rcp_ftz(d.y)});
    p[i] = fma2(move, both(-r.rate), mul2(p[i], both(r.decay)));
    ma = fmaxf(ma, fmaxf(fabsf(m[i].x), fabsf(m[i].y)));
    top = max(top, max(__float_as_uint(root[i].x), __float_as_uint(root[i].y)));     // a gradient that voids m voids v too
  }
  top = __reduce_max_sync(0xffffffffu, top);                        // by their bits: what is not finite lies above all else
  const bool finite = top < 0x7f800000u;
  if (!finite) {                                                    // rare: scales from the finite values alone
    ma = 0.f;
    top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float& me = i & 1 ? m[i >> 1].y : m[i >> 1].x;
      float& re = i & 1 ? root[i >> 1].y : root[i >> 1].x;
      if (fabsf(me) < INFINITY && re < INFINITY) {
        ma = fmaxf(ma, fabsf(me));
        top = max(top, __float_as_uint(re));
      } else {
        me = re = NAN;
        by_dither &= ~(1u << i);
      }
    }
    top = __reduce_max_sync(0xffffffffu, top);
  }
  // moments of 1e-30 and less are zero: their scale's reciprocal would overflow
  float mm = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(ma))), rm = __uint_as_float(top);
  mm = mm > 1e-30f ? mm : 0.f;
  rm = rm > kNoRoot ? rm : 0.f;
  sc = make_float2(mm * (1.f / 448.f), rm * (1.f / 448.f));
  const Pair mi = both(mm > 0.f ? rcp_ftz(sc.x) : 0.f), ri = both(rm > 0.f ? rcp_ftz(sc.y) : 0.f), ms = both(-sc.x), rs = both(-sc.y);
  uint32_t mw[4], vw[4], low = 0xffffffffu;
  Pair y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    Pair x = divide2(m[i], ms, mi);
    if constexpr (LOOK) {
      const uint32_t bits = mix(~(pair + i), r.step);
      if (by_dither >> (2 * i) & 1) x.x = copysignf(dithered(fabsf(x.x), ((bits & 0xffffu) << 4) | 8u), x.x);
      if (by_dither >> (2 * i) & 2) x.y = copysignf(dithered(fabsf(x.y), ((bits >> 16) << 4) | 8u), x.y);
    }
    mw[i] = __nv_cvt_float2_to_fp8x2(make_float2(x.x, x.y), __NV_SATFINITE, __NV_E4M3);
    y[i] = divide2(root[i], rs, ri);
    low = min(low, min(__float_as_uint(y[i].x), __float_as_uint(y[i].y)));
  }
  mc = make_uint2(mw[0] | (mw[1] << 16), mw[2] | (mw[3] << 16));
  if (finite && low >= 0x3c800000u) {
    // All of the thread's y lie at 2^-6 or above: a code is its fp32 bits 20 to 26 after the dither and less the exponents' distance
    // (120 << 23).  Times 16 they are the top byte: u * 16 + (dither * 16 - (120 << 27)), the latter put together from bytes.
    // The largest dither is 8 short of a code's distance, and the largest y some 3 ulps above 448: never the code beyond, a NaN.
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t bits = mix(pair + i, r.step);
      const uint32_t d0 = __byte_perm(bits, 0x00004080u, 0x5104), d1 = __byte_perm(bits, 0x00004080u, 0x5324);
      h[i] = __byte_perm(__float_as_uint(y[i].x) * 16u + d0, __float_as_uint(y[i].y) * 16u + d1, 0x0073);
    }
    vc = make_uint2(__byte_perm(h[0], h[1], 0x5410), __byte_perm(h[2], h[3], 0x5410));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t bits = mix(pair + i, r.step);
      float a = root[i].x > kNoRoot ? fmaxf(dithered(y[i].x, ((bits & 0xffffu) << 4) | 8u), 0x1p-9f) : 0.f;
      float b = root[i].y > kNoRoot ? fmaxf(dithered(y[i].y, ((bits >> 16) << 4) | 8u), 0x1p-9f) : 0.f;
      if (isnan(root[i].x)) a = NAN;
      if (isnan(root[i].y)) b = NAN;
      vw[i] = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    }
    vc = make_uint2(vw[0] | (vw[1] << 16), vw[2] | (vw[3] << 16));
  }
}

template <typename TP, typename TG, int BITS, bool MASTER, int N>
__global__ void __launch_bounds__(kThreads, 4)
adamw_kernel(const __grid_constant__ Table<N> table, const States st, const Rule r) {
  griddep_wait();
  griddep_launch_dependents();
  // The tensor of this chunk: the last one whose first chunk is not beyond it, from a coarse index and a search between two of its
  // entries (each step waits for the one before; one warp searching for all, behind a barrier, cost 8 %).
  const int chunk = blockIdx.x;
  int lo = table.near[chunk >> table.shift], hi = table.near[(chunk >> table.shift) + 1];
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (table.first[mid] <= chunk) lo = mid;
    else hi = mid - 1;
  }
  const TP* p = static_cast<const TP*>(table.p[lo]);
  const TG* g = static_cast<const TG*>(table.g[lo]);
  TP* out = static_cast<TP*>(table.out[lo]);
  const long long numel = table.numel[lo], at = table.at[lo];
  const bool p_vec = ((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  const bool g_vec = (reinterpret_cast<uintptr_t>(g) & 15) == 0;
  const float grad_scale = r.grad_scale_ptr != nullptr ? r.grad_scale * *r.grad_scale_ptr : r.grad_scale;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long from = static_cast<long long>(chunk - table.first[lo]) * kChunk<BITS>, to = min(from + kChunk<BITS>, numel);

  constexpr int kTimes = kRound / kThreads / 8;
  if constexpr (BITS == 8) {
    const long long start = from;
    using TV = std::conditional_t<MASTER, float, TP>;               // what holds the value: the parameter or its master
    // `whole`: every element of the chunk exists and every address is aligned, so nothing is asked per lane (3 instructions an
    // element less); else lanes past the end load nothing and write nothing but the states' padding
    auto chunk_of = [&](auto whole_t) {
      constexpr bool whole = decltype(whole_t)::value;
      Raw8<TG> gr[kTimes];
      Raw8<TV> pr[kTimes];
      uint2 mc[kTimes], vc[kTimes];
      float2 sc[kTimes];
      const long long i0 = start + threadIdx.x * 8, j0 = at + i0;   // warp w has block w, then block w + 8
      const TG* gp = g + i0;
      const TV* pp = MASTER ? reinterpret_cast<const TV*>(st.master + j0) : reinterpret_cast<const TV*>(p + i0);
      const uint8_t* mp = static_cast<const uint8_t*>(st.m) + j0;
      const uint8_t* vp = static_cast<const uint8_t*>(st.v) + j0;
      const long long b0 = (at + start) / kBlock + warp;
      auto left = [&](int it) { return numel - start - (it * (kThreads / 32) + warp) * kBlock; };   // elements from the warp's block on
      auto mine = [&](int it) { return whole ? 8 : static_cast<int>(min(max(left(it) - lane * 8, 0ll), 8ll)); };
#pragma unroll
      for (int it = 0; it < kTimes; ++it) {                         // all loads first
        if (!whole && left(it) <= 0) continue;                      // uniform in the warp
        constexpr int kStep = kThreads * 8;
        fetch8(gp + it * kStep, whole || g_vec, mine(it), gr[it]);
        fetch8(pp + it * kStep, whole || MASTER || p_vec, MASTER ? 8 : mine(it), pr[it]);
        mc[it] = __ldcs(reinterpret_cast<const uint2*>(mp + it * kStep));
        vc[it] = __ldcs(reinterpret_cast<const uint2*>(vp + it * kStep));
        sc[it] = st.scales[b0 + it * (kThreads / 32)];
      }
      TP* op = out + i0;
#pragma unroll
      for (int it = 0; it < kTimes; ++it) {
        if (!whole && left(it) <= 0) continue;
        constexpr int kStep = kThreads * 8;
        Pair gv[4], pv[4];
        unpack(gr[it], gv);
        if (grad_scale != 1.f)
#pragma unroll
          for (int i = 0; i < 4; ++i) gv[i] = mul2(gv[i], both(grad_scale));
        unpack(pr[it], pv);
        const uint32_t pair = static_cast<uint32_t>(j0 >> 1) + it * (kStep / 2);
        // top bit of a byte: the old code's exponent is not zero, so m is 2^-6 or more
        constexpr uint32_t kExp = 0x78787878u, kTop = 0x80808080u;
        const uint32_t normal = ((mc[it].x & kExp) + kExp) & ((mc[it].y & kExp) + kExp) & kTop;
        if (__any_sync(0xffffffffu, normal != kTop || r.dither_m)) step8<true>(mc[it], vc[it], sc[it], gv, pv, r, pair);
        else step8<false>(mc[it], vc[it], sc[it], gv, pv, r, pair);
        const float flat[8] = {pv[0].x, pv[0].y, pv[1].x, pv[1].y, pv[2].x, pv[2].y, pv[3].x, pv[3].y};
        if constexpr (MASTER) store8(st.master_out + j0 + it * kStep, true, 8, flat);
        store8(op + it * kStep, whole || p_vec, mine(it), flat);
        __stcs(reinterpret_cast<uint2*>(static_cast<uint8_t*>(st.m_out) + j0 + it * kStep), mc[it]);
        __stcs(reinterpret_cast<uint2*>(static_cast<uint8_t*>(st.v_out) + j0 + it * kStep), vc[it]);
        if (lane == 0) st.scales_out[b0 + it * (kThreads / 32)] = sc[it];
      }
    };
    if (start + kRound <= numel && p_vec && g_vec) chunk_of(std::true_type{});
    else chunk_of(std::false_type{});
  } else {
#pragma unroll 1
    for (long long start = from; start < to; start += kRound)
#pragma unroll
    for (int it = 0; it < kTimes; ++it) {
      const long long block = start + (it * (kThreads / 32) + warp) * kBlock;
      if (block >= numel) break;
      const long long i = block + lane * 8, j = at + i;
      const int n = static_cast<int>(min(max(numel - i, 0ll), 8ll));
      float pv[8], gv[8], m[8], v[8];
      load8(g + i, g_vec, n, gv);
      if constexpr (MASTER) load8(st.master + j, true, 8, pv);
      else load8(p + i, p_vec, n, pv);
      load8(static_cast<const float*>(st.m) + j, true, 8, m);
      load8(static_cast<const float*>(st.v) + j, true, 8, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float a = gv[e] * grad_scale;
        m[e] = fmaf(r.beta1, m[e], r.one_beta1 * a);
        v[e] = fmaf(r.beta2, v[e], r.one_beta2 * a * a);
        pv[e] = fmaf(pv[e], r.decay, -r.rate * __fdividef(m[e], fmaf(sqrtf(v[e]), r.root, r.eps)));
      }
      if constexpr (MASTER) {
        if (n < 8) {                                                // padding stays zero, which 0 / (0 + eps) is not without an eps
#pragma unroll
          for (int e = 0; e < 8; ++e) pv[e] = e < n ? pv[e] : 0.f;
        }
        store8(st.master_out + j, true, 8, pv);
      }
      store8(out + i, p_vec, n, pv);
      store8(static_cast<float*>(st.m_out) + j, true, 8, m);
      store8(static_cast<float*>(st.v_out) + j, true, 8, v);
    }
  }
}

template <typename TP, typename TG, int BITS, bool MASTER, int N>
int launch_n(const b200tp_adamw_tensor* t, int count, const States& st, const Rule& r, cudaStream_t stream) {
  Table<N> table;
  int chunks = 0, kept = 0;
  for (int i = 0; i < count; ++i) {
    if (t[i].numel == 0) continue;
    table.p[kept] = t[i].param;
    table.g[kept] = t[i].grad;
    table.out[kept] = t[i].param_out;
    table.numel[kept] = t[i].numel;
    table.at[kept] = t[i].state_offset;
    table.first[kept++] = chunks;
    chunks += static_cast<int>(ceil_div(t[i].numel, kChunk<BITS>));
  }
  if (kept == 0) return B200TP_OK;
  table.first[kept] = chunks;
  table.shift = 0;
  while (((chunks - 1) >> table.shift) >= kNear) ++table.shift;
  for (int k = 0, i = 0; k <= kNear; ++k) {
    while (i + 1 < kept && table.first[i + 1] <= static_cast<int64_t>(k) << table.shift) ++i;
    table.near[k] = static_cast<short>(i);
  }
  B200TP_CUDA_OK(launch_pdl(adamw_kernel<TP, TG, BITS, MASTER, N>, dim3(chunks), dim3(kThreads), 0, stream, table, st, r));
  return B200TP_OK;
}

// Few tensors to a launch: by their number, and by their chunks so that the grid and `first` stay in 31 bits.
template <typename TP, typename TG, int BITS, bool MASTER>
int launch_all(const b200tp_adamw_tensor* t, int count, const States& st, const Rule& r, cudaStream_t stream) {
  int i = 0;
  while (i < count) {
    int n = 0;
    int64_t chunks = 0;
    while (i + n < count && n < kTensors && (n == 0 || chunks + ceil_div(t[i + n].numel, kChunk<BITS>) < (1ll << 31) - 1))
      chunks += ceil_div(t[i + n++].numel, kChunk<BITS>);
    const int rc = n <= kFew ? launch_n<TP, TG, BITS, MASTER, kFew>(t + i, n, st, r, stream)
                             : launch_n<TP, TG, BITS, MASTER, kTensors>(t + i, n, st, r, stream);
    if (rc) return rc;
    i += n;
  }
  return B200TP_OK;
}

template <typename TP, typename TG>
int launch_kind(const b200tp_adamw_args* a, const b200tp_adamw_tensor* t, int count, const States& st, const Rule& r,
                cudaStream_t stream) {
  if constexpr (sizeof(TP) == 2) {
    if (a->master != nullptr)
      return a->bits == 8 ? launch_all<TP, TG, 8, true>(t, count, st, r, stream) : launch_all<TP, TG, 32, true>(t, count, st, r, stream);
  }
  return a->bits == 8 ? launch_all<TP, TG, 8, false>(t, count, st, r, stream) : launch_all<TP, TG, 32, false>(t, count, st, r, stream);
}

bool misaligned(const void* p, unsigned mask) { return (reinterpret_cast<uintptr_t>(p) & mask) != 0; }

// Written ranges that overlap, or overlap what another tensor's step reads, would race: the same tensor twice, views of one another, an
// output over another tensor's input or gradient.
using Ranges = std::vector<std::pair<uintptr_t, uintptr_t>>;
int check_apart(Ranges& ranges, const char* what) {
  std::sort(ranges.begin(), ranges.end());
  for (size_t i = 1; i < ranges.size(); ++i)
    if (ranges[i].first < ranges[i - 1].second)
      return fail(B200TP_ERR_OPTIM_INPUT, std::string("two tensors of one step share memory (") + what + ")");
  return B200TP_OK;
}

int check(const b200tp_adamw_args* a, const b200tp_adamw_tensor* t, int32_t count) {
  if (a == nullptr || (t == nullptr && count > 0)) return fail(B200TP_ERR_OPTIM_INPUT, "args or the tensors are null");
  if (count < 0) return fail(B200TP_ERR_OPTIM_INPUT, "negative number of tensors");
  if ((a->param_dtype != B200TP_F32 && a->param_dtype != B200TP_BF16) || (a->grad_dtype != B200TP_F32 && a->grad_dtype != B200TP_BF16))
    return fail(B200TP_ERR_OPTIM_INPUT, "parameters and gradients must be fp32 or bf16");
  if (a->bits != 8 && a->bits != 32) return fail(B200TP_ERR_OPTIM_INPUT, "moments are kept in 8 or 32 bits");
  if ((a->master == nullptr) != (a->master_out == nullptr)) return fail(B200TP_ERR_OPTIM_INPUT, "master and master_out go together");
  if (a->master != nullptr && a->param_dtype == B200TP_F32) return fail(B200TP_ERR_OPTIM_INPUT, "fp32 parameters need no masters");
  if (a->step < 1) return fail(B200TP_ERR_OPTIM_INPUT, "step counts from 1");
  if (!(a->beta1 >= 0. && a->beta1 < 1.) || !(a->beta2 >= 0. && a->beta2 < 1.)) return fail(B200TP_ERR_OPTIM_INPUT, "betas must lie in [0, 1)");
  if (!(a->eps >= 0.) || !(a->lr >= 0.) || !(a->weight_decay >= 0.))
    return fail(B200TP_ERR_OPTIM_INPUT, "lr, eps and weight_decay must not be negative");
  const bool some = std::any_of(t, t + count, [](const b200tp_adamw_tensor& x) { return x.numel != 0; });
  if (some && (a->exp_avg == nullptr || a->exp_avg_sq == nullptr || a->exp_avg_out == nullptr || a->exp_avg_sq_out == nullptr ||
               (a->bits == 8 && (a->scales == nullptr || a->scales_out == nullptr))))
    return fail(B200TP_ERR_OPTIM_INPUT, "null states");
  const void* states[] = {a->exp_avg, a->exp_avg_sq, a->scales, a->master, a->exp_avg_out, a->exp_avg_sq_out, a->scales_out, a->master_out};
  for (const void* p : states)
    if (misaligned(p, 15)) return fail(B200TP_ERR_OPTIM_INPUT, "states must be 16-byte aligned");
  Ranges outs, inputs, offsets;
  outs.reserve(count);
  offsets.reserve(count);
  const unsigned p_item = a->param_dtype == B200TP_BF16 ? 2 : 4, g_item = a->grad_dtype == B200TP_BF16 ? 2 : 4;
  for (int i = 0; i < count; ++i) {
    if (t[i].numel < 0 || t[i].numel > (1ll << 42)) return fail(B200TP_ERR_OPTIM_INPUT, "bad number of elements");
    if (t[i].numel == 0) continue;
    if (t[i].param == nullptr || t[i].grad == nullptr || t[i].param_out == nullptr) return fail(B200TP_ERR_OPTIM_INPUT, "null tensor");
    if (misaligned(t[i].param, p_item - 1) || misaligned(t[i].param_out, p_item - 1) || misaligned(t[i].grad, g_item - 1))
      return fail(B200TP_ERR_OPTIM_INPUT, "a tensor is not aligned to its elements");
    if (t[i].state_offset < 0 || t[i].state_offset % kBlock != 0)
      return fail(B200TP_ERR_OPTIM_INPUT, "a tensor's place in the states must be a multiple of 256 elements");
    const uintptr_t p = reinterpret_cast<uintptr_t>(t[i].param_out), q = reinterpret_cast<uintptr_t>(t[i].param);
    outs.emplace_back(p, p + static_cast<uintptr_t>(t[i].numel) * p_item);
    if (q != p && a->master == nullptr) inputs.emplace_back(q, q + static_cast<uintptr_t>(t[i].numel) * p_item);
    offsets.emplace_back(t[i].state_offset, t[i].state_offset + align_up(t[i].numel, kBlock));
  }
  int rc = check_apart(outs, "parameters");
  if (rc) return rc;
  for (int i = 0; i < count; ++i) {           // a gradient may lie where its own results go, element on element
    if (t[i].numel == 0) continue;
    const uintptr_t g = reinterpret_cast<uintptr_t>(t[i].grad), end = g + static_cast<uintptr_t>(t[i].numel) * g_item;
    if (t[i].grad == t[i].param_out && g_item == p_item) continue;
    const auto next = std::lower_bound(outs.begin(), outs.end(), std::make_pair(end, uintptr_t{0}));    // begins behind it
    if (next != outs.begin() && std::prev(next)->second > g)
      return fail(B200TP_ERR_OPTIM_INPUT, "two tensors of one step share memory (a gradient and a parameter)");
  }
  if (!inputs.empty()) {
    inputs.insert(inputs.end(), outs.begin(), outs.end());
    rc = check_apart(inputs, "parameters");
    if (rc) return rc;
  }
  return check_apart(offsets, "states");
}

}  // namespace
}  // namespace b200tp

using namespace b200tp;

extern "C" int b200tp_adamw_step(const b200tp_adamw_args* a, const b200tp_adamw_tensor* tensors, int32_t count, void* stream_v) {
  try {
    int rc = check(a, tensors, count);
    if (rc) return rc;
    if (count == 0 || a->check_only != 0) return B200TP_OK;
    rc = require_sm100();
    if (rc) return rc;
    Rule r;
    r.beta1 = static_cast<float>(a->beta1);
    r.beta2 = static_cast<float>(a->beta2);
    r.one_beta1 = static_cast<float>(1. - a->beta1);
    r.one_beta2 = static_cast<float>(1. - a->beta2);
    r.eps = static_cast<float>(a->eps);
    r.decay = static_cast<float>(1. - a->lr * a->weight_decay);
    r.rate = static_cast<float>(a->lr / (1. - std::pow(a->beta1, static_cast<double>(a->step))));
    r.root = static_cast<float>(1. / std::sqrt(1. - std::pow(a->beta2, static_cast<double>(a->step))));
    r.grad_scale = static_cast<float>(a->grad_scale);
    r.grad_scale_ptr = a->grad_scale_ptr;
    r.step = static_cast<unsigned>(a->step);
    r.dither_m = a->beta1 > 0.9;
    States st;
    st.m = a->exp_avg;
    st.v = a->exp_avg_sq;
    st.scales = static_cast<const float2*>(a->scales);
    st.master = a->master;
    st.m_out = a->exp_avg_out;
    st.v_out = a->exp_avg_sq_out;
    st.scales_out = static_cast<float2*>(a->scales_out);
    st.master_out = a->master_out;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
    if (a->param_dtype == B200TP_BF16)
      return a->grad_dtype == B200TP_BF16 ? launch_kind<__nv_bfloat16, __nv_bfloat16>(a, tensors, count, st, r, stream)
                                          : launch_kind<__nv_bfloat16, float>(a, tensors, count, st, r, stream);
    return a->grad_dtype == B200TP_BF16 ? launch_kind<float, __nv_bfloat16>(a, tensors, count, st, r, stream)
                                        : launch_kind<float, float>(a, tensors, count, st, r, stream);
  } catch (const std::exception& e) {
    return fail(B200TP_ERR_OPTIM_INPUT, std::string("adamw: ") + e.what());
  }
}
