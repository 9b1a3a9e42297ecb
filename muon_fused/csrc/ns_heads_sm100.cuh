// Per-head Newton-Schulz in Gram form.
//
// A head is a block of d <= 128 rows (or columns) of a projection, n long, and
// is orthogonalised by itself.  With X0 = G/(‖G‖+1e-7) and A0 = X0·X0ᵀ (d x d),
// every iterate is a polynomial of A0 times X0, X_k = Q_k·X0, so the iteration
// runs on d x d matrices alone:
//
//   B = a·I + b·A + c·A²      Q ← B·Q      A ← B·A·B      (Q_0 = I)
//
// G is read for A0 and once more for Q·G; the whole-matrix path reads and
// writes X in each of its 15 products and pads every d-row block to a
// 256-row tile.  Three kernels:
//
//   heads_gram     G·Gᵀ, n split over a cluster               (HBM bound)
//   heads_iterate  norm and all iterations, a CTA per head    (latency bound)
//   heads_apply    out = Q·G/(‖G‖+1e-7)                       (HBM bound)
//
// Precision.  A0 is an fp32 sum of exact products.  Products of the 16-bit
// factors alone would not do: an error e in A0 grows by a² = 11.9 per step
// relative to a small eigenvalue, and single fp16 (bf16) factors leave 6-33 %
// (more) error in the result on ill-conditioned heads.  So A, B, C = B·A and Q
// are kept as fp16 pairs hi + lo (22 bits) and each product is three tensor-core
// products hi·hi + hi·lo + lo·hi in one fp32 accumulator; A is held scaled by
// DP so that its average diagonal is 1 and lo stays clear of fp16's subnormals.
// Q enters the last product as two terms of G's type.  The result is then within
// its bf16 rounding of the exact one for Gaussian and ill-conditioned (1e5) heads.
// What leaks into directions that a head does not span still grows by a² a step in A
// and from there by a in Q: with rank 8, 4, 2, 1 of 128 the error after 5 steps is
// 0.2, 0.25, 0.4, 0.7 %, after 6 already twice that and after 8 anything, so
// steps <= 5 (a third term of Q in the last product changed none of these).
//
// d is padded to DP = 64 or 128 by TMA's zero fill; padded rows and columns of A
// stay zero and change nothing.  tcgen05.mma always runs M = 128 here: with DP =
// 64 its upper 64 rows read whatever follows in shared memory and land in
// accumulator rows nobody reads.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

#include "fm_ptx.cuh"
#include "muon_elementwise.cuh"
#include "ns_gemm_sm100.cuh"
#include "ns_prep.cuh"

namespace fm {

// 4-D tile load: (inner, outer, head, matrix).
__device__ __forceinline__ void tma_load_4d(void* smem_dst, const CUtensorMap* map, uint64_t* bar,
                                            int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
__device__ __forceinline__ void tma_store_4d(const CUtensorMap* map, const void* smem_src, int c0,
                                             int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::
          "l"(reinterpret_cast<uint64_t>(map)),
      "r"(smem_u32(smem_src)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

// Instruction descriptor of kind::f16 with both operands fp16 (`half`) or bf16.
__host__ __device__ constexpr uint32_t make_idesc_16(bool half, int M, int N, int a_mn, int b_mn) {
  return half ? make_idesc_bf16(M, N, a_mn, b_mn) & ~((7u << 7) | (7u << 10))
              : make_idesc_bf16(M, N, a_mn, b_mn);
}

constexpr int kHeadsMaxDim = 128;
constexpr int kHeadsMaxSteps = 5;
constexpr int kHeadsK = 64;        // reduction columns per gram stage (one swizzle row)
constexpr int kGramMaxSplit = 8;   // portable cluster size
constexpr int kGramThreads = 192;  // producer, MMA, 4 epilogue warps
constexpr int kApplyN = 128;       // long-side elements per apply unit
constexpr int kApplyStages = 3;
constexpr int kApplyThreads = 320; // 8 epilogue warps, producer, MMA

// Index of element (row 32q + lane, col) in a stored DP x DP fp32 partial: a
// warp's access to one column is 128 contiguous bytes.
template <int DP>
__device__ __forceinline__ int gram_index(int q, int col, int lane) {
  return (q * DP + col) * 32 + lane;
}

// 16 bytes of another cluster CTA's shared memory.
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t cluster_addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(cluster_addr)
               : "memory");
  return v;
}

struct HeadsArgs {
  int d, n;          // head side, long side
  int heads;         // per matrix
  int total;         // heads x matrices
  int kblocks;       // ceil(n / kHeadsK)
  int split, kbps;   // gram: splits per head, k-blocks per split
  int steps;
  float* gram;       // total x DP x DP
  void* q;           // per head two terms of G's type, in the MMAs' swizzled layout
  float* inv;        // total: 1/(‖G‖+1e-7)
  __nv_bfloat16* out;
  long long out_ld, out_head, out_mat;  // strides of out: row, head, matrix (elements)
  int chunks;        // apply: ceil(n / kApplyN)
  int tma_out;
  unsigned* err;
};

// ------------------------------------------------------------------- gram
template <int DP>
struct GramCfg {
  // Two CTAs an SM for DP = 128, four for 64.
  static constexpr int kStages = DP == 128 ? 6 : 5;
  static constexpr int kStage = DP * kHeadsK * 2;
  // MMAs of M = 128 on DP = 64 read one stage past the last
  static constexpr int kSmem = (kStages + (DP == 64 ? 1 : 0)) * kStage + 1024 + 256;
  static_assert(DP * DP * 4 <= kStages * kStage, "the fp32 partial reuses the stages");
};

// A cluster of g.split CTAs per head, each with a range of n; its CTAs then add
// one share of the matrix each, in the order of the splits, from all CTAs' shared
// memory.  (Partials through global memory cost the iterate kernel, one CTA a
// head, 4 µs of reading at four splits.)
// COLS: heads are column blocks (the head side is contiguous in memory), so the
// operands are MN-major: a stage holds 64 long-side rows of DP columns.
template <int DP, bool COLS, bool HALF>
__global__ void __launch_bounds__(kGramThreads)
    heads_gram_kernel(const __grid_constant__ CUtensorMap tm, const HeadsArgs g) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  constexpr int kStage = GramCfg<DP>::kStage, kStages = GramCfg<DP>::kStages;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + (kStages + (DP == 64 ? 1 : 0)) * kStage);
  uint64_t* empty = full + kStages;
  uint64_t* acc_bar = empty + kStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(acc_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tm);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, DP);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();

  const int unit = blockIdx.x;
  const int head = unit / g.split, sp = unit - head * g.split;
  const int kb0 = sp * g.kbps, kb1 = min(g.kblocks, kb0 + g.kbps);
  const int h = head % g.heads, mat = head / g.heads;
  if (warp == 0) {
    if (lane == 0) {
      for (int kb = kb0; kb < kb1; ++kb) {
        const int i = kb - kb0, s = i % kStages;
        if (!mbar_wait(&empty[s], ((i / kStages) & 1) ^ 1, abort_flag, g.err, kErrWaitEmpty))
          break;
        mbar_arrive_expect_tx(&full[s], kStage);
        uint8_t* dst = smem + s * kStage;
        if constexpr (COLS) {
#pragma unroll
          for (int c = 0; c < DP / 64; ++c)
            tma_load_4d(dst + c * (kHeadsK * 128), &tm, &full[s], c * 64, kb * kHeadsK, h, mat);
        } else {
          tma_load_4d(dst, &tm, &full[s], kb * kHeadsK, 0, h, mat);
        }
      }
      pdl_trigger();
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = make_idesc_16(HALF, 128, DP, COLS ? 1 : 0, COLS ? 1 : 0);
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        const int i = kb - kb0, s = i % kStages;
        if (!mbar_wait(&full[s], (i / kStages) & 1, abort_flag, g.err, kErrWaitFull)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t base = smem_u32(smem + s * kStage);
#pragma unroll
        for (int k = 0; k < kHeadsK / 16; ++k) {
          // MN-major: 16 long-side rows are 2048 bytes, 64-column chunks 8 KB apart
          const uint64_t desc = COLS ? make_sdesc_sw128(base + k * 2048, kHeadsK * 128, 1024)
                                     : make_sdesc_sw128(base + k * 32, 16, 1024);
          tc_mma_bf16(tmem, desc, desc, idesc, (i | k) != 0 ? 1u : 0u);
        }
        tc_commit(&empty[s]);
      }
      if (ok) tc_commit(acc_bar);
    }
  } else {
    const int q = warp & 3;
    if (q * 32 < DP && mbar_wait(acc_bar, 0, abort_flag, g.err, kErrWaitAccFull)) {
      tc_fence_after();
      // the stages are free: every load has been consumed by a completed MMA
      float* dst = g.split == 1 ? g.gram + static_cast<long long>(head) * (DP * DP)
                                : reinterpret_cast<float*>(smem);
#pragma unroll 1
      for (int c = 0; c < DP / 32; ++c) {
        float v[32];
        tmem_ld_32x32b_x32(tmem + c * 32 + (static_cast<uint32_t>(q * 32) << 16), v);
#pragma unroll
        for (int k = 0; k < 32; ++k) dst[gram_index<DP>(q, c * 32 + k, lane)] = v[k];
      }
      tc_fence_before();
    }
    __syncwarp();
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, DP);
  }
  if (g.split > 1) {
    cluster_sync();  // every CTA's partial is in its shared memory
    const uint32_t base = smem_u32(smem);
    float4* dst = reinterpret_cast<float4*>(g.gram + static_cast<long long>(head) * (DP * DP));
    for (int i = sp * kGramThreads + threadIdx.x; i < DP * DP / 4; i += g.split * kGramThreads) {
      float4 x[kGramMaxSplit];  // all fetched before the first is added
#pragma unroll
      for (int s = 0; s < kGramMaxSplit; ++s)
        if (s < g.split) x[s] = ld_cluster_f4(mapa_shared(base + i * 16, s));
#pragma unroll
      for (int s = 1; s < kGramMaxSplit; ++s) {
        if (s < g.split) {
          x[0].x += x[s].x;
          x[0].y += x[s].y;
          x[0].z += x[s].z;
          x[0].w += x[s].w;
        }
      }
      __stcg(dst + i, x[0]);
    }
    cluster_sync();  // nobody leaves while its partial is read
  }
}

// ---------------------------------------------------------------- iterate
// One CTA per head.  With P = b·A + c·A² (the diagonal a·I stays in fp32):
//
//   A² → P      C = a·A + P·A      Q ← a·Q + P·Q      A ← a·C + P·C
//
// P is the MMAs' first factor in TMEM, A (then C in its place) and Q the second in
// shared memory, all as hi and lo.  The fp32 terms a·X and b·A are where the
// accumulators start: the epilogue that holds X writes them to TMEM before the
// product's MMAs, which all accumulate.  The tensor pipe sets the pace (24 MMAs of
// 64 clocks a product, 4 products an iteration); Q's product runs under C's
// epilogue and Q's epilogue under A², P's epilogue gives its columns in two halves
// so that C's MMAs start under the second, and A's is exposed.
//
// Measured at 128 x 128: 49-54k clocks for five iterations, 26k of them MMAs; the
// rest are P's epilogue (1k an iteration), hand-overs between the roles (0.4k each)
// and shared memory shared by MMAs and epilogues.
//
// Tried: hi alone for A² and P in the last iteration: 1 % faster, but the cut-off
// hi doubles the error of the result (3.2e-3 against 1.66e-3).  A CTA pair per head
// with cta_group::2 M = 128 (64 rows a CTA, two heads an SM): its MMAs took as long
// as M = 128 on one CTA, and arrivals at the peer's barrier cost more than the
// halved epilogue saved (330 against 326 µs on 384 heads of 128 x 4096).
constexpr int kIterWarps = 16;                        // epilogue warps
constexpr int kIterThreads = 32 * (kIterWarps + 1);   // and the MMA issuer

template <int DP>
struct IterCfg {
  static constexpr int kMat = DP * DP * 2;  // one 16-bit matrix: DP/64 k-blocks of DP rows
  static constexpr int kPer = DP / 8;       // columns per epilogue thread in each half
  static constexpr int kWarps = 4 * (DP / 32);  // epilogue warps with rows to hold
  static constexpr int kTmem = DP == 128 ? 512 : 256;  // 3 accumulators, P hi and lo
  static constexpr int kSmem = 4 * kMat + 1024 + 256;  // A and Q as hi and lo
};

// Packed fp32 pairs: one instruction for two lanes of an epilogue that the issue
// rate bounds.
__device__ __forceinline__ void mul2(float& x, float& y, float f) {
  asm("{\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %2};\n\t"
      "mul.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(f));
}
__device__ __forceinline__ void sub2(float& x, float& y, float u, float w) {
  asm("{\n\t.reg .b64 a, b, m;\n\t"
      "mov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\tmov.b64 m, {%4, %4};\n\t"
      "fma.rn.f32x2 a, b, m, a;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(u), "f"(w), "f"(-1.f));
}

// Two floats as packed 16-bit hi (returned) and the rest as packed lo.  fp16's hi
// is cut off in the float's bits (11 of them, so hi + lo has 22): converting it
// back from fp16 to subtract took as long as the rest of an epilogue.
template <bool HALF>
__device__ __forceinline__ uint32_t split2(float x, float y, uint32_t& lo) {
  if constexpr (HALF) {
    const float hx = __uint_as_float(__float_as_uint(x) & 0xffffe000u);
    const float hy = __uint_as_float(__float_as_uint(y) & 0xffffe000u);
    const __half2 h = __floats2half2_rn(hx, hy);
    sub2(x, y, hx, hy);
    const __half2 l = __floats2half2_rn(x, y);
    lo = *reinterpret_cast<const uint32_t*>(&l);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    const float2 f = __bfloat1622float2(h);
    const __nv_bfloat162 l = __floats2bfloat162_rn(x - f.x, y - f.y);
    lo = *reinterpret_cast<const uint32_t*>(&l);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// Hi and lo of 8 consecutive values into the swizzled K-major operand: row r,
// columns 8·chunk.. of k-block kb.
template <int DP, bool HALF = true>
__device__ __forceinline__ void put_split8(uint8_t* hi, int r, int kb, int chunk, const float* v) {
  const int off = kb * (DP * 128) + r * 128 + ((chunk ^ (r & 7)) << 4);
  uint4 h, l;
  h.x = split2<HALF>(v[0], v[1], l.x);
  h.y = split2<HALF>(v[2], v[3], l.y);
  h.z = split2<HALF>(v[4], v[5], l.z);
  h.w = split2<HALF>(v[6], v[7], l.w);
  *reinterpret_cast<uint4*>(hi + off) = h;
  *reinterpret_cast<uint4*>(hi + IterCfg<DP>::kMat + off) = l;
}

// 32 lanes x N consecutive 32-bit columns.
template <int N>
__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, float* v) {
  static_assert(N == 16 || N == 8);
  if constexpr (N == 16) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]),
          "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]),
          "=f"(v[14]), "=f"(v[15])
        : "r"(taddr)
        : "memory");
  } else {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]),
                   "=f"(v[6]), "=f"(v[7])
                 : "r"(taddr)
                 : "memory");
  }
}
// Completes this warp's loads; v's values are read after it.
template <int N>
__device__ __forceinline__ void tmem_wait_ld(float* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int k = 0; k < N; ++k) asm volatile("" : "+f"(v[k]));
}
template <int N>
__device__ __forceinline__ void tmem_st_cols(uint32_t taddr, const uint32_t* r) {
  static_assert(N == 8 || N == 4);
  if constexpr (N == 8) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
        : "memory");
  } else {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" ::"r"(taddr),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3])
                 : "memory");
  }
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// D[tmem] (+)= A[tmem] * B[smem]^T: lane = row of A, two 16-bit K elements a column.
__device__ __forceinline__ void tc_mma_16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc,
                                             uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Untiled bulk copies (both addresses and the size multiples of 16 bytes).
__device__ __forceinline__ void bulk_store(void* dst, const void* smem_src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst),
               "r"(smem_u32(smem_src)), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void bulk_load(void* smem_dst, const void* src, uint32_t bytes,
                                          uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          smem_u32(smem_dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

// DP = 64: two heads an SM (56 registers a thread do, and half the TMEM): 512 heads of
// 64 x 4096 237 -> 216 µs, 256 of 64 x 512 48 -> 38 µs, a few heads as before.
template <int DP, bool HALF>
__global__ void __launch_bounds__(kIterThreads, DP == 64 ? 2 : 1) heads_iterate_kernel(const HeadsArgs g) {
  using Cfg = IterCfg<DP>;
  constexpr int kPer = Cfg::kPer;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* sA = smem;  // hi, lo
  uint8_t* sQ = smem + 2 * Cfg::kMat;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + 4 * Cfg::kMat);
  uint64_t* op_a = bars;        // operand A (or C in its place) written
  uint64_t* op_c = bars + 1;
  uint64_t* op_p = bars + 2;    // [2]: P's column halves (and Q before them) written
  uint64_t* acc_sq = bars + 4;  // A² ready
  uint64_t* acc_c = bars + 5;   // P·A
  uint64_t* acc_q = bars + 6;   // P·Q
  uint64_t* acc_a = bars + 7;   // P·C
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* s_done = reinterpret_cast<int*>(tmem_slot + 2);    // Q staged by every epilogue warp
  float* s_tr = reinterpret_cast<float*>(tmem_slot + 4);  // trace, one part per epilogue warp
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int head = blockIdx.x;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 4; ++i) mbar_init(&bars[i], Cfg::kWarps);
    for (int i = 4; i < 8; ++i) mbar_init(&bars[i], 1);
    *abort_flag = 0;
    *s_done = 0;
    fence_barrier_init();
  }
  if (warp == kIterWarps) {
    tmem_alloc(tmem_slot, Cfg::kTmem);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t d0 = tmem, d1 = tmem + DP, d2 = tmem + 2 * DP;
  const uint32_t p_hi = tmem + 3 * DP, p_lo = p_hi + DP / 2;
  pdl_wait();
  pdl_trigger();

  // Epilogue warp: accumulator rows 32q.. and, of each half of the columns, kPer
  // from sub·kPer.
  const int q = warp & 3, sub = (warp >> 2) & 3;
  const int row = q * 32 + lane, col0 = sub * kPer;
  const bool worker = warp < kIterWarps && q * 32 < DP;
  const uint32_t lanes = static_cast<uint32_t>(q * 32) << 16;
  // A is held as A' = DP·A, so P = c/DP² · (b·DP/c · A' + A'²)
  constexpr float kScale = static_cast<float>(DP);
  constexpr float kP = kNsC / (kScale * kScale), kPA = kNsB * kScale / kNsC;
  float v[2][kPer];  // this thread's part of the matrix at hand
  if (worker) {
    const float* src = g.gram + static_cast<long long>(head) * (DP * DP);
    float tr = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int k = 0; k < kPer; ++k)
        v[h][k] = __ldcg(src + gram_index<DP>(q, h * (DP / 2) + col0 + k, lane));
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int k = 0; k < kPer; ++k) tr += h * (DP / 2) + col0 + k == row ? v[h][k] : 0.f;
    }
    tr = warp_sum(tr);
    if (lane == 0) s_tr[warp] = tr;
  }
  __syncthreads();

  if (worker) {
    float tr = 0.f;
#pragma unroll
    for (int w = 0; w < kIterWarps; ++w) tr += (w & 3) * 32 < DP ? s_tr[w] : 0.f;
    const float inv = 1.f / (sqrtf(tr) + 1e-7f);
    if (threadIdx.x == 0) g.inv[head] = inv;

    auto put = [&](uint8_t* dst, int h) {  // a half of v into an operand
      const int c = h * (DP / 2) + col0;
#pragma unroll
      for (int i = 0; i < kPer / 8; ++i)
        put_split8<DP>(dst, row, c / 64, (c % 64) / 8 + i, v[h] + 8 * i);
    };
    auto get = [&](uint32_t d) {  // v from an accumulator
      tc_fence_after();
      tmem_ld_cols<kPer>(d + col0 + lanes, v[0]);
      tmem_ld_cols<kPer>(d + DP / 2 + col0 + lanes, v[1]);
      tmem_wait_ld<kPer>(v[0]);
      tmem_wait_ld<kPer>(v[1]);
    };
    auto start = [&](uint32_t d, int h, float f) {  // f·v where an accumulator starts
#pragma unroll
      for (int i = 0; i < kPer / 8; ++i) {
        uint32_t r[8];
#pragma unroll
        for (int k = 0; k < 8; k += 2) {
          float x = v[h][8 * i + k], y = v[h][8 * i + k + 1];
          mul2(x, y, f);
          r[k] = __float_as_uint(x);
          r[k + 1] = __float_as_uint(y);
        }
        tmem_st_cols<8>(d + h * (DP / 2) + col0 + 8 * i + lanes, r);
      }
    };
    auto ready = [&](uint64_t* bar) {
      tmem_wait_st();
      tc_fence_before();
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    auto add_diag = [&](float f) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int k = 0; k < kPer; ++k)
          if (h * (DP / 2) + col0 + k == row) v[h][k] += f;
    };
    bool ok = true;
    if (g.steps == 0) {  // Q = I
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int k = 0; k < kPer; ++k) v[h][k] = 0.f;
      add_diag(1.f);
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        // inv twice: inv² alone may leave fp32's range where A does not
#pragma unroll
        for (int k = 0; k < kPer; ++k) v[h][k] = v[h][k] * inv * (inv * kScale);
        put(sA, h);
        start(d0, h, kPA);
        start(d1, h, kNsA);
      }
      ready(op_a);
    }
#pragma unroll 1
    for (int it = 0; it < g.steps; ++it) {
      const bool last = it == g.steps - 1;
      const uint32_t ph = it & 1;
      if (!(ok = mbar_wait(acc_sq, ph, abort_flag, g.err, kErrWaitAccFull))) break;
      get(d0);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t hi[kPer / 2], lo[kPer / 2];
#pragma unroll
        for (int k = 0; k < kPer / 2; ++k) {
          mul2(v[h][2 * k], v[h][2 * k + 1], kP);
          hi[k] = split2<true>(v[h][2 * k], v[h][2 * k + 1], lo[k]);
        }
        const uint32_t at = (h * (DP / 2) + col0) / 2 + lanes;
        tmem_st_cols<kPer / 2>(p_hi + at, hi);
        tmem_st_cols<kPer / 2>(p_lo + at, lo);
        if (it > 0 || !last) ready(op_p + h);
      }
      if (it == 0) {  // Q = a·I + P
        add_diag(kNsA);
        if (last) break;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          put(sQ, h);
          start(d2, h, kNsA);
        }
      }
      if (!last) {
        if (!(ok = mbar_wait(acc_c, ph, abort_flag, g.err, kErrWaitAccFull))) break;
        get(d1);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          put(sA, h);
          start(d0, h, kNsA);
        }
        ready(op_c);
        if (!(ok = mbar_wait(acc_a, ph, abort_flag, g.err, kErrWaitAccFull))) break;
        get(d0);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          put(sA, h);
          start(d0, h, kPA);
          start(d1, h, kNsA);
        }
        ready(op_a);
      }
      if (it > 0) {
        if (!(ok = mbar_wait(acc_q, ph ^ 1, abort_flag, g.err, kErrWaitAccFull))) break;
        get(d2);
        if (!last) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            put(sQ, h);
            start(d2, h, kNsA);
          }
        }
      }
    }
    if (ok) {
      // Q as two terms of G's type, staged in the layout that heads_apply's MMAs
      // read and copied out as it is.  Every product is complete.
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = h * (DP / 2) + col0;
#pragma unroll
        for (int i = 0; i < kPer / 8; ++i)
          put_split8<DP, HALF>(sQ, row, c / 64, (c % 64) / 8 + i, v[h] + 8 * i);
      }
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) {
        __threadfence_block();
        if (atomicAdd(s_done, 1) == Cfg::kWarps - 1) {
          __threadfence_block();
          fence_proxy_async_shared();
          bulk_store(static_cast<uint8_t*>(g.q) + static_cast<long long>(head) * (2 * Cfg::kMat), sQ,
                     2 * Cfg::kMat);
          bulk_commit();
          bulk_wait_all();
        }
      }
      __syncwarp();
    }
    tc_fence_before();
  } else if (warp == kIterWarps && lane == 0) {
    // The second factor is read MN-major, so that a product is X·Y and not X·Yᵀ:
    // beside the untransposed a·X terms, transposed ones would turn the antisymmetric
    // part of A's rounding error round in sign and let it grow by (2a - 1) a step.
    constexpr uint32_t idesc = make_idesc_16(true, 128, DP, 0, 1);
    constexpr int kSteps = DP / 16;  // K steps of a product
    auto first = [](uint32_t base, int k) {  // rows, 16 columns from 16·k
      return make_sdesc_sw128(base + (k / 4) * (DP * 128) + (k % 4) * 32, 16, 1024);
    };
    auto second = [](uint32_t base, int k) {  // 16 rows from 16·k, all columns
      return make_sdesc_sw128(base + k * 2048, DP * 128, 1024);
    };
    // D += P·Y over K steps [k0, k1): terms hi·hi + hi·lo + lo·hi.
    auto times_p = [&](uint32_t d, const uint8_t* y, int k0, int k1) {
      const uint32_t yb = smem_u32(y);
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        if (k < k0 || k >= k1) continue;
        const uint64_t yh = second(yb, k), yl = second(yb + Cfg::kMat, k);
        tc_mma_16_ts(d, p_hi + k * 8, yh, idesc, 1u);
        tc_mma_16_ts(d, p_hi + k * 8, yl, idesc, 1u);
        tc_mma_16_ts(d, p_lo + k * 8, yh, idesc, 1u);
      }
    };
    for (int it = 0; it < g.steps; ++it) {
      const bool last = it == g.steps - 1;
      const uint32_t ph = it & 1;
      if (!mbar_wait(op_a, ph, abort_flag, g.err, kErrWaitFull)) break;
      tc_fence_after();
      {
        const uint32_t ab = smem_u32(sA);
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          const uint64_t xh = first(ab, k), yh = second(ab, k);
          tc_mma_bf16(d0, xh, yh, idesc, 1u);
          tc_mma_bf16(d0, xh, second(ab + Cfg::kMat, k), idesc, 1u);
          tc_mma_bf16(d0, first(ab + Cfg::kMat, k), yh, idesc, 1u);
        }
      }
      tc_commit(acc_sq);
      if (it == 0 && last) break;
      const uint8_t* y = last ? sQ : sA;  // C, or the last step's Q
      const uint32_t d = last ? d2 : d1;
      if (!mbar_wait(&op_p[0], ph, abort_flag, g.err, kErrWaitFull)) break;
      tc_fence_after();
      times_p(d, y, 0, kSteps / 2);
      if (!mbar_wait(&op_p[1], ph, abort_flag, g.err, kErrWaitFull)) break;
      tc_fence_after();
      times_p(d, y, kSteps / 2, kSteps);
      if (last) {
        tc_commit(acc_q);
        break;
      }
      tc_commit(acc_c);
      if (it > 0) times_p(d2, sQ, 0, kSteps / 2);
      if (!mbar_wait(op_c, ph, abort_flag, g.err, kErrWaitFull)) break;
      tc_fence_after();
      times_p(d0, sA, 0, kSteps);
      tc_commit(acc_a);
      if (it > 0) {
        times_p(d2, sQ, kSteps / 2, kSteps);
        tc_commit(acc_q);
      }
    }
  }
  __syncthreads();
  if (warp == kIterWarps) {
    tc_fence_after();
    tmem_dealloc(tmem, Cfg::kTmem);
  }
}

// ------------------------------------------------------------------ apply
template <int DP>
struct ApplyCfg {
  // CTAs an SM.  Two at 64, where one has half the rows to write and the loads in
  // flight did not cover memory's latency (512 heads of 64 x 4096: 216 -> 193 µs,
  // with the gram kernel's four); at 128 shared memory holds one.
  static constexpr int kCtas = DP == 128 ? 1 : 2;
  static constexpr int kStage = DP * kApplyN * 2;
  static constexpr int kQ = 2 * DP * DP * 2;            // both terms of one head
  static constexpr int kWriters = DP / 16;              // epilogue warps with output
  static constexpr int kStaging = kWriters * 32 * 64 * 2 * 2;  // two 32 x 64 blocks each
  // MMAs of M = 128 on DP = 64 read 8 KB past Q, which the staging covers
  static constexpr int kSmem = kApplyStages * kStage + kQ + kStaging + 1024 + 256;
};

// Stores one staged 32 x 64 bf16 block (128-byte rows, 16-byte chunks XORed
// with row & 7) element by element, four rows fetched before they are written
// (4 x (4096, 4091): 193 -> 175 µs).  Aligned pairs instead, with a row's odd ends apart,
// took 285: the three ways of a warp through each row cost more than the stores.
__device__ __forceinline__ void store_block_plain(const uint8_t* blk, __nv_bfloat16* dst,
                                                  long long ld, int rows, int cols, int lane) {
  const unsigned short* src = reinterpret_cast<const unsigned short*>(blk);
  unsigned short* to = reinterpret_cast<unsigned short*>(dst) + lane;
#pragma unroll 1
  for (int r0 = 0; r0 < rows; r0 += 4, to += 4 * ld) {
    unsigned short x[4][2];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int p = 0; p < 2; ++p)
        x[r][p] = src[(r0 + r) * 64 + ((((lane >> 3) + 4 * p) ^ ((r0 + r) & 7)) << 3) + (lane & 7)];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int p = 0; p < 2; ++p)
        if (r0 + r < rows && p * 32 + lane < cols) to[r * ld + p * 32] = x[r][p];
  }
}

// Units are (head, chunk of 128 long-side elements), walked by contiguous
// ranges so that a block loads a head's Q once or twice.  Row heads: D = Q·G
// (rows of the head x 128 columns).  Column heads: D = G·Q (128 rows x columns
// of the head), Q being symmetric.
template <int DP, bool COLS, bool HALF>
__global__ void __launch_bounds__(kApplyThreads, ApplyCfg<DP>::kCtas)
    heads_apply_kernel(const __grid_constant__ CUtensorMap tmG,
                       const __grid_constant__ CUtensorMap tmO, const HeadsArgs g) {
  using Cfg = ApplyCfg<DP>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* sG = smem;
  uint8_t* sQ = smem + kApplyStages * Cfg::kStage;
  uint8_t* staging = sQ + Cfg::kQ;
  uint64_t* full = reinterpret_cast<uint64_t*>(staging + Cfg::kStaging);
  uint64_t* empty = full + kApplyStages;
  uint64_t* q_full = empty + kApplyStages;
  uint64_t* q_empty = q_full + 1;
  uint64_t* accf = q_empty + 1;  // [2]
  uint64_t* acce = accf + 2;     // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acce + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kAccWarps = COLS ? 8 : 2 * (DP / 32);  // epilogue warps that drain an accumulator

  if (threadIdx.x == 0) {
    for (int s = 0; s < kApplyStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&accf[s], 1);
      mbar_init(&acce[s], kAccWarps);
    }
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmG);
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 256);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  const long long units = static_cast<long long>(g.total) * g.chunks;
  const long long u0 = units * blockIdx.x / gridDim.x, u1 = units * (blockIdx.x + 1) / gridDim.x;

  if (warp == 8) {
    // producer
    if (lane == 0) {
      int head_in = -1;
      uint32_t q_phase = 0;
      int i = 0;
      pdl_wait();
      for (long long u = u0; u < u1; ++u, ++i) {
        const int head = static_cast<int>(u / g.chunks), chunk = static_cast<int>(u % g.chunks);
        const int h = head % g.heads, mat = head / g.heads;
        if (head != head_in) {
          if (!mbar_wait(q_empty, q_phase ^ 1, abort_flag, g.err, kErrWaitEmpty)) break;
          mbar_arrive_expect_tx(q_full, Cfg::kQ);
          bulk_load(sQ, static_cast<const uint8_t*>(g.q) + static_cast<long long>(head) * Cfg::kQ,
                    Cfg::kQ, q_full);
          q_phase ^= 1;
          head_in = head;
        }
        const int s = i % kApplyStages;
        if (!mbar_wait(&empty[s], ((i / kApplyStages) & 1) ^ 1, abort_flag, g.err, kErrWaitEmpty))
          break;
        mbar_arrive_expect_tx(&full[s], Cfg::kStage);
        uint8_t* dst = sG + s * Cfg::kStage;
        if constexpr (COLS) {
#pragma unroll
          for (int c = 0; c < DP / 64; ++c)
            tma_load_4d(dst + c * (kApplyN * 128), &tmG, &full[s], c * 64, chunk * kApplyN, h, mat);
        } else {
#pragma unroll
          for (int c = 0; c < kApplyN / 64; ++c)
            tma_load_4d(dst + c * (DP * 128), &tmG, &full[s], chunk * kApplyN + c * 64, 0, h, mat);
        }
      }
    }
  } else if (warp == 9) {
    // MMA issuer
    if (lane == 0) {
      constexpr uint32_t idesc = COLS ? make_idesc_16(HALF, 128, DP, 0, 0)
                                      : make_idesc_16(HALF, 128, kApplyN, 0, 1);
      int head_in = -1;
      uint32_t q_phase = 0;
      int i = 0;
      for (long long u = u0; u < u1; ++u, ++i) {
        const int head = static_cast<int>(u / g.chunks);
        if (head != head_in) {
          // the previous head's MMAs have read its Q once they complete
          if (head_in >= 0) tc_commit(q_empty);
          if (!mbar_wait(q_full, q_phase, abort_flag, g.err, kErrWaitFull)) break;
          q_phase ^= 1;
          head_in = head;
        }
        const int acc = i & 1, s = i % kApplyStages;
        if (!mbar_wait(&acce[acc], ((i >> 1) & 1) ^ 1, abort_flag, g.err, kErrWaitAccEmpty)) break;
        if (!mbar_wait(&full[s], (i / kApplyStages) & 1, abort_flag, g.err, kErrWaitFull)) break;
        tc_fence_after();
        const uint32_t gb = smem_u32(sG + s * Cfg::kStage), qb = smem_u32(sQ);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
          for (int k = 0; k < DP / 16; ++k) {
            const uint64_t qd = make_sdesc_sw128(
                qb + t * (DP * DP * 2) + (k / 4) * (DP * 128) + (k % 4) * 32, 16, 1024);
            const uint32_t first = (t | k) != 0 ? 1u : 0u;
            if constexpr (COLS) {
              const uint64_t gd =
                  make_sdesc_sw128(gb + (k / 4) * (kApplyN * 128) + (k % 4) * 32, 16, 1024);
              tc_mma_bf16(tmem + acc * 128, gd, qd, idesc, first);
            } else {
              // MN-major: 16 head rows are 2048 bytes, 64-column chunks DP rows apart
              const uint64_t gd = make_sdesc_sw128(gb + k * 2048, DP * 128, 1024);
              tc_mma_bf16(tmem + acc * 128, qd, gd, idesc, first);
            }
          }
        }
        tc_commit(&empty[s]);
        tc_commit(&accf[acc]);
      }
    }
  } else {
    // epilogue: rows 32q.. of the accumulator, columns 64·(warp / 4)..
    const int q = warp & 3, half = warp >> 2;
    const bool worker = COLS ? half * 64 < DP : q * 32 < DP;
    pdl_wait();
    if (worker || COLS) {
      // writers are numbered by lane quarter, then column half
      const int writer = half * (COLS ? 4 : DP / 32) + q;
      uint8_t* buf = staging + (worker ? writer : 0) * (32 * 64 * 2 * 2);
      int i = 0;
      // Blocks that this warp wrote.  The two buffers alternate by it and not by the unit:
      // a warp whose block lies past the matrix's end skips a unit, and the store of the
      // unit before is then the newest one, which the wait below lets go on reading.
      int written = 0;
      for (long long u = u0; u < u1; ++u, ++i) {
        const int head = static_cast<int>(u / g.chunks), chunk = static_cast<int>(u % g.chunks);
        const int h = head % g.heads, mat = head / g.heads;
        const int acc = i & 1;
        // the block's place in the output: rows r0.., columns c0.. of the head
        const int r0 = COLS ? chunk * kApplyN + q * 32 : q * 32;
        const int c0 = COLS ? half * 64 : chunk * kApplyN + half * 64;
        const int rows = min(32, (COLS ? g.n : g.d) - r0), cols = min(64, (COLS ? g.d : g.n) - c0);
        const float inv = __ldcg(g.inv + head);
        if (!mbar_wait(&accf[acc], (i >> 1) & 1, abort_flag, g.err, kErrWaitAccFull)) break;
        tc_fence_after();
        const bool any = worker && rows > 0 && cols > 0;
        uint8_t* blk = buf + (written & 1) * (32 * 64 * 2);
        if (any) {
          ++written;
          if (g.tma_out) {
            if (lane == 0) bulk_wait_read<1>();  // the block written before the last has been read
            __syncwarp();
          }
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float v[32];
            tmem_ld_32x32b_x32(
                tmem + acc * 128 + half * 64 + c * 32 + (static_cast<uint32_t>(q * 32) << 16), v);
#pragma unroll
            for (int k = 0; k < 32; k += 2) mul2(v[k], v[k + 1], inv);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              *reinterpret_cast<uint4*>(blk + lane * 128 + (((4 * c + k) ^ (lane & 7)) << 4)) =
                  pack8_bf16(v + 8 * k);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acce[acc]);
        if (any) {
          if (g.tma_out) {
            fence_proxy_async_shared();
            __syncwarp();
            if (lane == 0) {
              tma_store_4d(&tmO, blk, c0, r0, h, mat);
              bulk_commit();
            }
          } else {
            store_block_plain(blk,
                              g.out + mat * g.out_mat + h * g.out_head + r0 * g.out_ld + c0,
                              g.out_ld, rows, cols, lane);
            __syncwarp();
          }
        }
      }
      if (lane == 0) bulk_wait_all();
      __syncwarp();
    }
  }
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 256);
  }
}

// ------------------------------------------------------------------- pack
// Copy of G that TMA can address, for inputs it cannot (other types, unaligned
// rows or heads): outer x inner blocks per head with a row stride of ld
// elements (a multiple of 8), values rounded to T.  A thread gathers eight
// elements and stores 16 bytes; padding columns are never read.
__device__ __forceinline__ float as_16(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float as_16(__half x) { return __half2float(x); }
__device__ __forceinline__ float as_16(float x) { return x; }
__device__ __forceinline__ float as_16(double x) { return __bfloat162float(__double2bfloat16(x)); }

constexpr int kPackThreads = 256;

// VEC: every row of every head starts on a 16-byte boundary and has whole chunks (fp32
// and fp64: 16-bit types are then read in place).  A kernel of its own, since its
// registers would cost the other form occupancy (bf16 of 4091 columns: 175 -> 184 µs).
template <typename S, typename T, bool VEC>
__global__ void __launch_bounds__(kPackThreads)
    heads_pack_kernel(const S* __restrict__ G, long long ldg, long long mat_stride, int heads,
                      long long head_stride, long long outer, int inner, T* __restrict__ dst,
                      int ld) {
  pdl_wait();
  const int head = blockIdx.y;
  const S* src = G + (head / heads) * mat_stride + (head % heads) * head_stride;
  uint4* out = reinterpret_cast<uint4*>(dst + head * outer * ld);
  const unsigned chunks = static_cast<unsigned>(ld) / 8;
  const long long n = outer * chunks;
  const long long stride = static_cast<long long>(gridDim.x) * kPackThreads;
  auto place = [&](long long i, int& c) {
    const long long r = n <= 0xffffffffll ? static_cast<unsigned>(i) / chunks : i / chunks;
    c = static_cast<int>(i - r * chunks) * 8;
    return src + r * ldg + c;
  };
  long long i = static_cast<long long>(blockIdx.x) * kPackThreads + threadIdx.x;
  if constexpr (VEC) {
    // 16-byte loads, two chunks in flight (4 x (4096, 4096): fp32 175 -> 169 µs, fp64
    // 240 -> 209); element by element two are slower than one (182 against 175)
    constexpr int kVec = 16 / static_cast<int>(sizeof(S));
    for (; i < n; i += 2 * stride) {
      __align__(16) S x[2][8];
      int c;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (i + u * stride >= n) break;
        const S* p = place(i + u * stride, c);
#pragma unroll
        for (int k = 0; k < 8; k += kVec)
          *reinterpret_cast<uint4*>(&x[u][k]) = __ldcs(reinterpret_cast<const uint4*>(p + k));
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (i + u * stride >= n) break;
        __align__(16) T v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = from_f<T>(as_16(x[u][k]));
        out[i + u * stride] = *reinterpret_cast<const uint4*>(v);
      }
    }
  } else {
    for (; i < n; i += stride) {
      int c;
      const S* p = place(i, c);
      __align__(16) T v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = from_f<T>(c + k < inner ? as_16(p[k]) : 0.f);
      out[i] = *reinterpret_cast<const uint4*>(v);
    }
  }
}

}  // namespace fm
