// AdamW over a list of tensors in one launch (the optimizer's AdamW branch,
// reference muon_fused/optimizer.py:165-200, nine torch ops per tensor there):
//
//   m = m + (1-b1)·(g - m)          v = v + (1-b2)·(g² - v)
//   p = p·(1 - lr·wd) + alpha · m / (eps + sqrt(v)),   alpha = -lr·sqrt(1-b2^t)/(1-b1^t)
//
// Every element is read and written once: 28 bytes in fp32, 22 with 16-bit
// parameters and fp32 moments.  HBM bounds long lists, the launch short ones.
//
// Rounding.  Where the moments have the parameter's type the result is the
// torch chain's bit for bit: one rounding to that type after each of its ops
// (square, lerp, sqrt, + eps, /, *, + alpha·), lerp and the alpha-scaled add as
// one fused multiply-add each.  16-bit parameters with fp32 moments (a state
// the torch chain never had) are computed in fp32 and rounded once.
//
// Layout.  The list travels as a kernel parameter (no copy to the device, so
// a captured graph holds it); each block finds its tensor by bisection over
// the first-chunk indices and handles one chunk of it.
#pragma once
#include <cstdint>

#include "muon_elementwise.cuh"

namespace fm {

constexpr int kAdamThreads = 256;
constexpr int kAdamUnits = 2;                                  // 4-element units per thread
constexpr int kAdamChunk = kAdamThreads * 4 * kAdamUnits;      // elements per block

struct AdamEntry {
  void* p;
  const void* g;
  void* m;
  void* v;
  long long n;
  float alpha;
  unsigned first;  // index of the tensor's first chunk in the launch
};

// Tensors per launch: a short table for short lists (its copy into the launch is
// what a small call pays for), a long one just under the 32764-byte parameter limit.
// The long table adds 3.4 µs to a call: 24 vectors of 4096 take 8.2 µs through the
// short one, 25 take 11.7 through the long one, 65 take 17.7 (fp32, host included).
constexpr int kAdamSmall = 24;
constexpr int kAdamLarge = 640;

template <int CAP>
struct AdamTable {
  AdamEntry e[CAP];
  int count;
  float decay, w1, w2, eps;
};

// torch's lerp: the form depends on the weight so that weight 1 is exact.
__device__ __forceinline__ float lerp_torch(float a, float b, float w) {
  const float d = __fsub_rn(b, a);
  return fabsf(w) < 0.5f ? fmaf(w, d, a) : fmaf(-d, __fsub_rn(1.f, w), b);
}

template <typename T, typename M>
__device__ __forceinline__ void adam1(float& p, float g, float& m, float& v, float alpha,
                                      float decay, float w1, float w2, float eps) {
  constexpr bool kChain = sizeof(T) == sizeof(M);  // the torch chain's types
  m = to_f(from_f<M>(lerp_torch(m, g, w1)));
  const float g2 = to_f(from_f<M>(__fmul_rn(g, g)));
  v = to_f(from_f<M>(lerp_torch(v, g2, w2)));
  const float s = to_f(from_f<M>(__fsqrt_rn(v)));
  const float d = to_f(from_f<M>(__fadd_rn(s, eps)));
  const float u = to_f(from_f<M>(__fdiv_rn(m, d)));
  float p1 = __fmul_rn(p, decay);
  if constexpr (kChain) p1 = to_f(from_f<T>(p1));
  p = fmaf(alpha, u, p1);
}

// Four consecutive elements, streamed (nothing here is read twice).
template <typename T>
__device__ __forceinline__ void load4(const T* p, float (&x)[4]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = __ldcs(reinterpret_cast<const float4*>(p));
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
  } else {
    const uint2 u = __ldcs(reinterpret_cast<const uint2*>(p));
    const T* h = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = to_f(h[k]);
  }
}

template <typename T>
__device__ __forceinline__ void store4(T* p, const float (&x)[4]) {
  if constexpr (sizeof(T) == 4) {
    __stcs(reinterpret_cast<float4*>(p), make_float4(x[0], x[1], x[2], x[3]));
  } else {
    uint2 u;
    T* h = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int k = 0; k < 4; ++k) h[k] = from_f<T>(x[k]);
    __stcs(reinterpret_cast<uint2*>(p), u);
  }
}

template <typename T, typename M, int CAP>
__global__ void __launch_bounds__(kAdamThreads)
    adamw_list_kernel(const __grid_constant__ AdamTable<CAP> t) {
  int lo = 0, hi = t.count;  // last entry whose first chunk is not past this block
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.e[mid].first <= blockIdx.x) lo = mid; else hi = mid;
  }
  const AdamEntry& e = t.e[lo];
  const long long off = static_cast<long long>(blockIdx.x - e.first) * kAdamChunk;
  const int n = static_cast<int>(min(static_cast<long long>(kAdamChunk), e.n - off));
  T* p = static_cast<T*>(e.p) + off;
  const T* g = static_cast<const T*>(e.g) + off;
  M* m = static_cast<M*>(e.m) + off;
  M* v = static_cast<M*>(e.v) + off;
  const float alpha = e.alpha;
  const bool vec = aligned16(p) && aligned16(g) && aligned16(m) && aligned16(v);
  if (vec && n == kAdamChunk) {
    float pv[kAdamUnits][4], gv[kAdamUnits][4], mv[kAdamUnits][4], vv[kAdamUnits][4];
#pragma unroll
    for (int u = 0; u < kAdamUnits; ++u) {
      const int i = (u * kAdamThreads + threadIdx.x) * 4;
      load4(g + i, gv[u]);
      load4(m + i, mv[u]);
      load4(v + i, vv[u]);
      load4(p + i, pv[u]);
    }
#pragma unroll
    for (int u = 0; u < kAdamUnits; ++u) {
      const int i = (u * kAdamThreads + threadIdx.x) * 4;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        adam1<T, M>(pv[u][k], gv[u][k], mv[u][k], vv[u][k], alpha, t.decay, t.w1, t.w2, t.eps);
      store4(m + i, mv[u]);
      store4(v + i, vv[u]);
      store4(p + i, pv[u]);
    }
  } else {
    for (int i = threadIdx.x; i < n; i += kAdamThreads) {
      float pv = to_f(p[i]), mv = to_f(m[i]), vv = to_f(v[i]);
      adam1<T, M>(pv, to_f(g[i]), mv, vv, alpha, t.decay, t.w1, t.w2, t.eps);
      p[i] = from_f<T>(pv);
      m[i] = from_f<M>(mv);
      v[i] = from_f<M>(vv);
    }
  }
}

}  // namespace fm
