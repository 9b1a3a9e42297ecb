// Decay + neuron-wise normalised update of same-shape matrices (rows = output
// neurons, u = the bf16 orthogonalised update):
//
//   s_i = mean_j u_ij²             v_i = b2·v_i + (1-b2)·s_i
//   r_i = 1 / (sqrt(v_i) + eps)    F = ‖diag(r)·u‖_F = sqrt(Σ_i cols·s_i·r_i²)
//   p_ij = p_ij·(1 - lr·wd) - lr·0.2·sqrt(rows·cols)/(F + 1e-7) · r_i · u_ij
//
// F needs only the row sums, so two passes over u and one over p suffice:
//   normed_rows   one row per warp (or block): Σ u², v, r and the block's share of F²
//   normed_scale  F from the shares; r_i becomes the row's whole factor of u
//   normed_apply  p, walking the matrix backwards so that the rows of u read
//                 last by normed_rows are still in L2
// normed_scale is a launch of its own (2 µs) because apply cannot afford it: with
// every apply block adding up the shares, that chain of loads and not HBM set the
// pace (107 against 53 µs on a bf16 4096 x 14336 matrix).
// The launches overlap where their data allow it (programmatic dependent launch):
// apply fetches its p and u before it waits for the factors, and the row pass of
// the next matrices runs while apply drains, waiting for it at its own end only, so
// that the end of the call is the end of all of it (6 bf16 4096 x 14336 matrices:
// 420 -> 409 µs; 5 fp32 1003 x 2731: 36 -> 33).  The call's first row pass waits at
// its start, before it lets anything follow: nothing here reads what an earlier
// kernel may still be writing.
// HBM bounds both passes.  All statistics are fp32; p is rounded once.  Sums run in
// a fixed order (no atomics), so results repeat bit for bit.
#pragma once
#include <cstdint>

#include "fm_ptx.cuh"
#include "adamw_list.cuh"
#include "muon_elementwise.cuh"
#include "ns_prep.cuh"

namespace fm {

constexpr int kNormedThreads = 256;
constexpr int kNormedList = 64;        // matrices per launch
constexpr int kNormedMaxBlocks = 16384;  // row blocks per matrix = shares of F² per matrix
constexpr int kNormedUnits = 4;        // apply: 4-element units per thread
constexpr int kNormedChunk = kNormedThreads * 4 * kNormedUnits;  // elements per apply block

struct NormedEntry {
  void* p;
  const __nv_bfloat16* u;
  float* v;
};

struct NormedArgs {
  NormedEntry e[kNormedList];
  long long rows, cols;
  float* rinv;      // rows floats per matrix
  float* partials;  // row_blocks per matrix
  int row_blocks;
  int first;        // the call's first row pass
  float decay, step, beta2, w2, eps;  // step = lr·0.2·sqrt(rows·cols), w2 = 1 - beta2
};

__device__ __forceinline__ float bf16x8_sumsq(uint4 u, float acc) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
    acc = fmaf(f.x, f.x, acc);
    acc = fmaf(f.y, f.y, acc);
  }
  return acc;
}

// Σ u² over one row by `width` threads (t = 0..width-1): elements up to the
// first 16-byte boundary, 16-byte loads, the rest.
__device__ __forceinline__ float row_sumsq(const __nv_bfloat16* row, long long cols, int t,
                                           int width) {
  const long long mis = (reinterpret_cast<uintptr_t>(row) & 15) / 2;
  const long long head = mis ? min(cols, 8 - mis) : 0;
  const long long vecs = (cols - head) / 8;
  const uint4* q = reinterpret_cast<const uint4*>(row + head);
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  long long i = t;
  for (; i + 3ll * width < vecs; i += 4ll * width) {
    uint4 a[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) a[k] = __ldg(q + i + static_cast<long long>(k) * width);
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[k] = bf16x8_sumsq(a[k], acc[k]);
  }
  {  // up to three more, fetched together
    uint4 a[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const long long j = i + static_cast<long long>(k) * width;
      a[k] = j < vecs ? __ldg(q + j) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) acc[k] = bf16x8_sumsq(a[k], acc[k]);
  }
  if (t < head) {
    const float x = __bfloat162float(row[t]);
    acc[1] = fmaf(x, x, acc[1]);
  }
  const long long tail = head + vecs * 8;
  if (tail + t < cols) {
    const float x = __bfloat162float(row[tail + t]);
    acc[2] = fmaf(x, x, acc[2]);
  }
  return (acc[0] + acc[1]) + (acc[2] + acc[3]);
}

// v, r and the share of F² of one row whose Σ u² is s (one thread).
__device__ __forceinline__ float normed_row(const NormedArgs& a, float* v, float* rinv, float v_old,
                                            float s) {
  // w2 comes from the host, rounded once: 1 - beta2 of a beta2 already rounded to fp32 is
  // off by 1.3e-5 at 0.999 and 1.7e-4 at 0.9999
  const float x = fmaf(a.beta2, v_old, a.w2 * (s / static_cast<float>(a.cols)));
  *v = x;
  const float ri = 1.f / (sqrtf(x) + a.eps);
  *rinv = ri;
  return s * ri * ri;
}

// TPR threads per row: a warp where a row is short, the block where it is long.
template <int TPR>
__global__ void __launch_bounds__(kNormedThreads, 6)
    normed_rows_kernel(const __grid_constant__ NormedArgs a) {
  constexpr int kWarps = kNormedThreads / 32;
  constexpr int kPer = kNormedThreads / TPR;  // rows per block and round
  __shared__ float s_part[kWarps];
  if (a.first) pdl_wait();
  pdl_trigger();
  const NormedEntry e = a.e[blockIdx.y];
  float* rinv = a.rinv + a.rows * blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = threadIdx.x / TPR, t = threadIdx.x % TPR;
  float f2 = 0.f;  // the share of F² of the rows that this thread finished
  for (long long r0 = static_cast<long long>(blockIdx.x) * kPer; r0 < a.rows;
       r0 += static_cast<long long>(gridDim.x) * kPer) {
    const long long r = r0 + sub;
    const bool ok = r < a.rows;
    const float v_old = ok && t == 0 ? e.v[r] : 0.f;  // fetched beside the row
    float s = warp_sum(ok ? row_sumsq(e.u + r * a.cols, a.cols, t, TPR) : 0.f);
    if constexpr (TPR > 32) {
      if (lane == 0) s_part[warp] = s;
      __syncthreads();
      if (threadIdx.x == 0) {
        s = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) s += s_part[w];
        f2 += normed_row(a, e.v + r, rinv + r, v_old, s);
      }
      if (r0 + static_cast<long long>(gridDim.x) * kPer < a.rows) __syncthreads();
    } else if (ok && lane == 0) {
      f2 += normed_row(a, e.v + r, rinv + r, v_old, s);
    }
  }
  if constexpr (TPR == 32) {
    if (lane == 0) s_part[warp] = f2;
    __syncthreads();
    if (threadIdx.x == 0) {
      f2 = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) f2 += s_part[w];
    }
  }
  if (threadIdx.x == 0)
    a.partials[static_cast<long long>(blockIdx.y) * a.row_blocks + blockIdx.x] = f2;
  if (!a.first) pdl_wait();
}

// -step / (F + 1e-7) from the shares of F², added by the whole block in one order.
__device__ __forceinline__ float normed_eta(const NormedArgs& a, float* s_part) {
  const float* part = a.partials + static_cast<long long>(blockIdx.y) * a.row_blocks;
  float f2 = 0.f;
  for (int i0 = 0; i0 < a.row_blocks; i0 += 8 * kNormedThreads) {
    float x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int i = i0 + k * kNormedThreads + threadIdx.x;
      x[k] = i < a.row_blocks ? part[i] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) f2 += x[k];
  }
  f2 = warp_sum(f2);
  if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = f2;
  __syncthreads();
  f2 = 0.f;
#pragma unroll
  for (int w = 0; w < kNormedThreads / 32; ++w) f2 += s_part[w];
  return -a.step / (sqrtf(f2) + 1e-7f);
}

// Turns r into -step/(F + 1e-7) · r.
__global__ void __launch_bounds__(kNormedThreads)
    normed_scale_kernel(const __grid_constant__ NormedArgs a) {
  __shared__ float s_part[kNormedThreads / 32];
  pdl_trigger();
  pdl_wait();
  float* rinv = a.rinv + a.rows * blockIdx.y;
  const float eta = normed_eta(a, s_part);
  for (long long r = static_cast<long long>(blockIdx.x) * kNormedThreads + threadIdx.x; r < a.rows;
       r += static_cast<long long>(gridDim.x) * kNormedThreads)
    rinv[r] *= eta;
}

// Four elements, the i-th.. of a chunk whose first row ends after `rem` elements
// of it: p = p·decay + eta·f·u, where f is the factor of each element's row.  The four
// lie in one row where cols divides by 4 (ROW4), else in two at most where a row
// has four elements.
template <bool ROW4>
__device__ __forceinline__ void normed4(float (&p)[4], const float (&u)[4], const float* r, int i,
                                        int rem, unsigned cols, float decay, float eta, int cnt) {
  float f[4];
  const unsigned past = static_cast<unsigned>(i - rem);
  const unsigned q = i < rem ? 0u : 1u + past / cols;
  if constexpr (ROW4) {
    f[0] = f[1] = f[2] = f[3] = r[q];
  } else if (cols >= 4) {
    const unsigned left = i < rem ? static_cast<unsigned>(rem - i) : cols - past % cols;
    const float f0 = r[q], f1 = left < static_cast<unsigned>(min(4, cnt)) ? r[q + 1] : f0;
#pragma unroll
    for (int k = 0; k < 4; ++k) f[k] = static_cast<unsigned>(k) < left ? f0 : f1;
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      f[k] = k < cnt ? r[i + k < rem ? 0u : 1u + static_cast<unsigned>(i + k - rem) / cols] : 0.f;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) p[k] = fmaf(eta * f[k], u[k], __fmul_rn(p[k], decay));
}

// One block per chunk of 4096 consecutive elements, the last chunk first.  FOLD:
// r is not scaled yet, and every block adds up the shares itself: for matrices of
// a few blocks an SM, where that chain costs less than the launch it replaces.
template <typename T, bool ROW4, bool FOLD>
__global__ void __launch_bounds__(kNormedThreads)
    normed_apply_kernel(const __grid_constant__ NormedArgs a) {
  __shared__ float s_part[kNormedThreads / 32];
  pdl_trigger();
  const NormedEntry e = a.e[blockIdx.y];
  const long long n = a.rows * a.cols;
  const long long e0 = static_cast<long long>(gridDim.x - 1 - blockIdx.x) * kNormedChunk;
  T* p = static_cast<T*>(e.p) + e0;
  const __nv_bfloat16* u = e.u + e0;
  // 32-bit division where it is enough: the 64-bit one costs as much as the chunk's arithmetic
  const long long r0 = n <= 0xffffffffll
                           ? static_cast<unsigned>(e0) / static_cast<unsigned>(a.cols)
                           : e0 / a.cols;
  // elements of the chunk in its first row, and a row's length, in 32 bits (a row
  // past that is longer than any chunk)
  const int rem = static_cast<int>(min((r0 + 1) * a.cols - e0, 0x7fffffffll));
  const unsigned cols = static_cast<unsigned>(min(a.cols, 0xffffffffll));
  const float* r = a.rinv + a.rows * blockIdx.y + r0;
  if (e0 + kNormedChunk <= n && aligned16(p) && aligned16(u)) {
    const bool one_row = rem >= kNormedChunk;  // the whole chunk
    float pv[kNormedUnits][4], uv[kNormedUnits][4];
#pragma unroll
    for (int w = 0; w < kNormedUnits; ++w) {
      load4(p + (w * kNormedThreads + threadIdx.x) * 4, pv[w]);
      load4(u + (w * kNormedThreads + threadIdx.x) * 4, uv[w]);
    }
    pdl_wait();
    float f = *r;
    const float eta = FOLD ? normed_eta(a, s_part) : 1.f;
    f *= eta;
#pragma unroll
    for (int w = 0; w < kNormedUnits; ++w) {
      const int i = (w * kNormedThreads + threadIdx.x) * 4;
      if (one_row) {
#pragma unroll
        for (int k = 0; k < 4; ++k) pv[w][k] = fmaf(f, uv[w][k], __fmul_rn(pv[w][k], a.decay));
      } else {
        normed4<ROW4>(pv[w], uv[w], r, i, rem, cols, a.decay, eta, 4);
      }
      store4(p + i, pv[w]);
    }
  } else {
    const int cnt = static_cast<int>(min(static_cast<long long>(kNormedChunk), n - e0));
    pdl_wait();
    const float eta = FOLD ? normed_eta(a, s_part) : 1.f;
    for (int i = threadIdx.x * 4; i < cnt; i += kNormedThreads * 4) {
      float pv[4], uv[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        pv[k] = i + k < cnt ? to_f(p[i + k]) : 0.f;
        uv[k] = i + k < cnt ? __bfloat162float(u[i + k]) : 0.f;
      }
      normed4<ROW4>(pv, uv, r, i, rem, cols, a.decay, eta, cnt - i);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i + k < cnt) p[i + k] = from_f<T>(pv[k]);
    }
  }
}

}  // namespace fm
