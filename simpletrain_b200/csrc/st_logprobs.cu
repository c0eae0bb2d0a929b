// Log probabilities of given tokens, entropies and top alternatives of rows of
// logits, with the gradient (C ABI in include/st_fused_ops.h).
//
// Mathematics, in base 2 so that each element costs one ex2: y = c * logit with
// c = log2(e) / temperature, m = max y, s = sum 2^(y-m), w = sum 2^(y-m) (y-m):
//   lse = ln2 (m + log2 s), kept in double for the gradient      logprob = ln2 (y_token - m - log2 s)
//   entropy = ln2 (log2 s - w / s)
//   dlogit_v = (a ([v = token] - p_v) - b p_v (ln p_v + entropy)) / temperature
// One pass over the row keeps a running (m, s, w) per thread, rescaled when a
// vector raises the maximum; the triples are merged across the block and, where
// a cluster of CTAs shares a row, across the cluster through distributed shared
// memory (no workspace, no atomics on global memory).
//
// Top alternatives: a thread's maximum over its elements comes out of the same
// pass.  The k-th largest of the block's thread maxima bounds the block's k-th
// largest element from below, so a second sweep (of L2: the row was just read)
// keeps only elements at or above it, a little over k of them, and ranks those by
// (value, then lowest index).  When more than kCand elements tie at or above the
// bound (constant rows, rows with fewer than k finite values) they are selected
// one by one instead, a sweep each.
//
// Measured, 16384 rows of 32000 in bf16: forward 182 us (5.8 TB/s, 0.89 of a copy's rate), gradient
// 330 us (6.4 TB/s, 0.98).  128 rows of 50257 in fp32 with 20 alternatives: 15.3 us (16.5 a call); one row of
// 32000 with 5: 7.4 us.  The gradient of a slice of wider rows, whose alignment the contiguous result does not share, goes
// element by element: 4096 rows of 50257 of 50304 in bf16 426 us against 147 us for contiguous ones.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/st_fused_ops.h"
#include "kda_internal.h"
#include "tc_common.cuh"

namespace cg = cooperative_groups;

namespace {

using kda::tc::pack2;
using kda::tc::unpack2;

constexpr int kBlock = 256;
constexpr int kWarps = kBlock / 32;
constexpr int kTopMax = 32;
constexpr int kCand = 1024;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr double kLog2eD = 1.4426950408889634, kLn2D = 0.6931471805599453;
// y - m below this contributes 2^-300 = 0 in fp32; a floor keeps 0 * (y - m) finite for y = -inf
constexpr float kFloor = -300.f;
// Logits below kStart are masked: probability 0 (the lowest values of bf16 and fp32 are).  The running
// maximum starts there, and masked logits count as kMask, whose distance to it is 2^-huge = 0; the
// two are far apart so that the rounding of c times them cannot turn that distance positive.
constexpr float kStart = -1.2345e29f;
constexpr float kMask = -1e30f;

enum { kBF16 = 0, kF16 = 1, kF32 = 2 };

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int DT>
struct Elem {
  static constexpr int kBytes = DT == kF32 ? 4 : 2;
  static constexpr int kVec = 16 / kBytes;
  static __device__ __forceinline__ float load(const char *row, int64_t i) {
    if (DT == kF32) return reinterpret_cast<const float *>(row)[i];
    return unpack2((uint32_t) reinterpret_cast<const uint16_t *>(row)[i], DT == kBF16).x;
  }
  static __device__ __forceinline__ void store(char *row, int64_t i, float v) {
    if (DT == kF32)
      reinterpret_cast<float *>(row)[i] = v;
    else
      reinterpret_cast<uint16_t *>(row)[i] = (uint16_t)(pack2(v, 0.f, DT == kBF16) & 0xffffu);
  }
  static __device__ __forceinline__ void unpack(const uint4 &v, float (&f)[kVec]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (DT == kF32) {
        f[i] = __uint_as_float(w[i]);
      } else {
        const float2 p = unpack2(w[i], DT == kBF16);
        f[2 * i] = p.x;
        f[(2 * i + 1) % kVec] = p.y;
      }
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[kVec]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (DT == kF32)
        w[i] = __float_as_uint(f[i]);
      else
        w[i] = pack2(f[2 * i], f[(2 * i + 1) % kVec], DT == kBF16);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// The largest of each half of a vector of 16-bit pairs (NaN if one is NaN)
template <int DT>
__device__ __forceinline__ uint32_t packed_max(const uint4 &v) {
  uint32_t a, b, m;
  if (DT == kBF16) {
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(a) : "r"(v.x), "r"(v.y));
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(b) : "r"(v.z), "r"(v.w));
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(b));
  } else {
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(a) : "r"(v.x), "r"(v.y));
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(b) : "r"(v.z), "r"(v.w));
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(b));
  }
  return m;
}

// Largest element of a 16-byte vector; NaN if one is NaN.
template <int DT>
__device__ __forceinline__ float vec_max(const uint4 &v) {
  if (DT == kF32) {
    float a, b;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(a) : "f"(__uint_as_float(v.x)), "f"(__uint_as_float(v.y)));
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(b) : "f"(__uint_as_float(v.z)), "f"(__uint_as_float(v.w)));
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(a) : "f"(a), "f"(b));
    return a;
  }
  const float2 p = unpack2(packed_max<DT>(v), DT == kBF16);
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(p.x), "f"(p.y));
  return r;
}

// Elements below kMask raised to it (NaN stays NaN): what a mask leaves (-inf, a type's lowest
// value) has probability 0, and 0 * (y - m) must be 0 and not NaN.  bf16 does that in pairs; fp16
// ends at -65504, which is a value like others, so it is done after the conversion.
__device__ __forceinline__ float floor1(float x, float low = kMask) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(low));
  return r;
}
template <int DT, int N>
__device__ __forceinline__ void unpack_floored(uint4 v, float (&f)[N]) {
  if (DT == kBF16) {
    auto pair = [](uint32_t &x) { asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(x) : "r"(x), "r"(0xF149F149u)); };
    pair(v.x);
    pair(v.y);
    pair(v.z);
    pair(v.w);
  }
  Elem<DT>::unpack(v, f);
  if (DT != kBF16)
#pragma unroll
    for (int k = 0; k < N; ++k) f[k] = floor1(f[k]);
}

// The part of a row that one CTA of the row's cluster owns: scalar elements
// [lo, body), 16-byte vectors from element `body`, scalar elements [tail, hi).
// Rows need only be element-aligned.
struct Slice {
  int64_t lo, body, nvec, tail, hi;
};

template <int DT>
__device__ __forceinline__ Slice slice_of(const char *row, int64_t V, int rank, int parts) {
  using E = Elem<DT>;
  const int64_t mis = (int64_t)(reinterpret_cast<uintptr_t>(row) & 15u) / E::kBytes;
  int64_t head = mis ? E::kVec - mis : 0;
  if (head > V) head = V;
  const int64_t nv = (V - head) / E::kVec;
  const int64_t v0 = nv * rank / parts, v1 = nv * (rank + 1) / parts;
  Slice s;
  s.body = head + v0 * E::kVec;
  s.nvec = v1 - v0;
  s.lo = rank == 0 ? 0 : s.body;
  s.tail = s.body + s.nvec * E::kVec;
  s.hi = rank == parts - 1 ? V : s.tail;
  return s;
}

// fn(index, value) for every element of the slice, spread over the block.
template <int DT, typename F>
__device__ __forceinline__ void for_each(const char *row, const Slice &sl, F fn) {
  using E = Elem<DT>;
  const uint4 *v4 = reinterpret_cast<const uint4 *>(row + sl.body * E::kBytes);
  for (int64_t i = threadIdx.x; i < sl.nvec; i += kBlock) {
    float f[E::kVec];
    E::unpack(__ldg(v4 + i), f);
#pragma unroll
    for (int k = 0; k < E::kVec; ++k) fn(sl.body + i * E::kVec + k, f[k]);
  }
  for (int64_t i = sl.lo + threadIdx.x; i < sl.body; i += kBlock) fn(i, E::load(row, i));
  for (int64_t i = sl.tail + threadIdx.x; i < sl.hi; i += kBlock) fn(i, E::load(row, i));
}

// running (m, s, w), m = c * (largest logit, kStart at least).  A row whose m never leaves c * kStart
// is empty.
struct Stat {
  float m, s, w;
};

__device__ __forceinline__ Stat merge(const Stat &a, const Stat &b) {
  const float M = fmaxf(a.m, b.m), da = fmaxf(a.m - M, kFloor), db = fmaxf(b.m - M, kFloor);
  const float fa = ex2(da), fb = ex2(db);
  return {M, a.s * fa + b.s * fb, (a.w + da * a.s) * fa + (b.w + db * b.s) * fb};
}

__device__ __forceinline__ void raise(Stat &t, float m) {
  const float d = fmaxf(t.m - m, kFloor), f = ex2(d);
  t.w = (t.w + d * t.s) * f;
  t.s *= f;
  t.m = m;
}

__device__ __forceinline__ void add1(Stat &t, float x, float c) {
  x = floor1(x);
  const float y = c * x;
  if (y > t.m) raise(t, y);
  const float d = fmaf(x, c, -t.m), e = ex2(d);  // (y - t.m would be off by y's rounding, as much as the exponents that count)
  t.s += e;
  t.w = fmaf(e, fmaxf(d, kFloor), t.w);
}

// Vectors of a slice that its threads keep in registers, so that the second sweep reads no memory.
constexpr int kKeep = 8;

// -infinity in every element
template <int DT>
__device__ __forceinline__ uint4 vec_nothing() {
  const uint32_t x = DT == kF32 ? 0xFF800000u : (DT == kBF16 ? 0xFF80FF80u : 0xFC00FC00u);
  return make_uint4(x, x, x, x);
}

template <int DT>
__device__ __forceinline__ uint4 vec_max2(const uint4 &a, const uint4 &b) {
  auto f = [](uint32_t x, uint32_t y) {
    uint32_t r;
    if (DT == kBF16)
      asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y));
    else if (DT == kF16)
      asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y));
    else
      asm("max.NaN.f32 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y));
    return r;
  };
  return make_uint4(f(a.x, b.x), f(a.y, b.y), f(a.z, b.z), f(a.w, b.w));
}

// F vectors into the running triple.  The maximum is looked after once for all of them: some lane of
// a warp raises it nearly every time, and the whole warp then pays for the rescaling.
template <int DT, int F, int N>
__device__ __forceinline__ void add_batch(Stat &t, const uint4 (&raw)[N], int first, float c) {
  using E = Elem<DT>;
  uint4 mv = raw[first];
#pragma unroll
  for (int j = 1; j < F; ++j) mv = vec_max2<DT>(mv, raw[first + j]);
  const float top = vec_max<DT>(mv), y = c * floor1(top);
  if (!(y <= t.m)) {  // a larger maximum, or a NaN
    if (y != y) {
      t.s = t.w = NAN;
      return;
    }
    raise(t, y);
  }
  float s0 = 0.f, s1 = 0.f, w0 = 0.f, w1 = 0.f;
#pragma unroll
  for (int j = 0; j < F; ++j) {
    float f[E::kVec];
    unpack_floored<DT>(raw[first + j], f);
#pragma unroll
    for (int k = 0; k < E::kVec; k += 2) {
      const float d0 = fmaf(f[k], c, -t.m), d1 = fmaf(f[k + 1], c, -t.m);
      const float e0 = ex2(d0), e1 = ex2(d1);
      s0 += e0;
      s1 += e1;
      w0 = fmaf(e0, d0, w0);
      w1 = fmaf(e1, d1, w1);
    }
  }
  t.s += s0 + s1;
  t.w += w0 + w1;
}

template <int DT>
__device__ __forceinline__ Stat sweep(const char *row, const Slice &sl, float c, uint4 (&keep)[kKeep], bool kept) {
  using E = Elem<DT>;
  Stat t{c * kStart, 0.f, 0.f};
  const uint4 *v4 = reinterpret_cast<const uint4 *>(row + sl.body * E::kBytes);
  const int n = (int)sl.nvec, tid = threadIdx.x;
  constexpr int F = 4;  // loads in flight a thread
  if (kept) {
#pragma unroll
    for (int j = 0; j < kKeep; ++j) keep[j] = tid + j * kBlock < n ? __ldg(v4 + tid + j * kBlock) : vec_nothing<DT>();
#pragma unroll
    for (int j = 0; j < kKeep; j += F)
      if (j * kBlock < n) add_batch<DT, F>(t, keep, j, c);
  } else {
    for (int i = tid; i < n; i += F * kBlock) {
      uint4 r[F];
#pragma unroll
      for (int j = 0; j < F; ++j) r[j] = i + j * kBlock < n ? __ldg(v4 + i + j * kBlock) : vec_nothing<DT>();
      add_batch<DT, F>(t, r, 0, c);
    }
  }
  for (int64_t j = sl.lo + threadIdx.x; j < sl.body; j += kBlock) add1(t, E::load(row, j), c);
  for (int64_t j = sl.tail + threadIdx.x; j < sl.hi; j += kBlock) add1(t, E::load(row, j), c);
  return t;
}

// (value, index) order: larger value first, then the lower index
__device__ __forceinline__ bool before(float va, int ia, float vb, int ib) { return va > vb || (va == vb && ia < ib); }
__device__ __forceinline__ float sort_key(float x) { return x == x ? x : -INFINITY; }

constexpr int kGroups = kBlock / 4;

struct Shared {
  Stat part[kWarps];
  Stat total;         // this CTA's
  float gmax[kGroups];
  float bound;
  int count;
  float cand_v[kCand];
  int cand_i[kCand];
  float top_v[kTopMax];  // this CTA's best k, in order
  int top_i[kTopMax];
  float red_v[kWarps];
  int red_i[kWarps];
};

// This CTA's best k of its slice into sh.top_*, in order; missing places get (-inf, INT_MAX).
// thread_max is the thread's largest c * logit (c > 0, and rounding keeps the order: a logit
// at or above the k-th largest has c * logit at or above the bound).  The bound is the k-th
// largest of the 64 maxima of four threads each: k <= 32 of them leave about 64 ln(64 / (64 -
// k)) candidates, 24 for k = 20, and ranking them costs a quarter of ranking all threads'.
template <int DT>
__device__ void local_top(const char *row, const Slice &sl, float c, float thread_max, int k, Shared &sh,
                          const uint4 (&keep)[kKeep], bool kept) {
  using E = Elem<DT>;
  const int tid = threadIdx.x;
  float gm = fmaxf(thread_max, __shfl_xor_sync(0xffffffffu, thread_max, 1));
  gm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, 2));
  if ((tid & 3) == 0) sh.gmax[tid >> 2] = gm;
  if (tid < kTopMax) {
    sh.top_v[tid] = -INFINITY;
    sh.top_i[tid] = 0x7fffffff;
  }
  if (tid == 0) sh.count = 0;
  __syncthreads();
  if (tid < kGroups) {
    const float mine = sh.gmax[tid];
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < kGroups; ++j) rank += before(sh.gmax[j], j, mine, tid) ? 1 : 0;
    if (rank == k - 1) sh.bound = mine;
  }
  __syncthreads();
  const float bound = sh.bound > c * kStart ? sh.bound : -INFINITY;  // fewer than k logits that are not masked
  auto offer = [&](int64_t i, float x) {
    x = sort_key(x);
    if (c * floor1(x) >= bound) {
      const int at = atomicAdd(&sh.count, 1);
      if (at < kCand) {
        sh.cand_v[at] = x;
        sh.cand_i[at] = (int)i;
      }
    }
  };
  auto offer_vec = [&](int64_t i, const uint4 &raw) {
    const float mv = vec_max<DT>(raw);
    if (c * floor1(mv) >= bound || mv != mv) {  // few vectors hold a candidate
      float f[E::kVec];
      E::unpack(raw, f);
#pragma unroll
      for (int e = 0; e < E::kVec; ++e) offer(sl.body + i * E::kVec + e, f[e]);
    }
  };
  if (kept) {
#pragma unroll
    for (int j = 0; j < kKeep; ++j)
      if (tid + j * kBlock < sl.nvec) offer_vec(tid + j * kBlock, keep[j]);
  } else {
    const uint4 *v4 = reinterpret_cast<const uint4 *>(row + sl.body * E::kBytes);
    constexpr int F = 8;  // loads in flight a thread
    for (int64_t i = tid; i < sl.nvec; i += F * kBlock) {
      uint4 r[F];
#pragma unroll
      for (int j = 0; j < F; ++j)
        if (i + j * kBlock < sl.nvec) r[j] = __ldg(v4 + i + j * kBlock);
#pragma unroll
      for (int j = 0; j < F; ++j)
        if (i + j * kBlock < sl.nvec) offer_vec(i + j * kBlock, r[j]);
    }
  }
  for (int64_t i = sl.lo + tid; i < sl.body; i += kBlock) offer(i, E::load(row, i));
  for (int64_t i = sl.tail + tid; i < sl.hi; i += kBlock) offer(i, E::load(row, i));
  __syncthreads();
  const int n = sh.count;
  if (n <= kCand) {
    for (int a = tid; a < n; a += kBlock) {
      const float v = sh.cand_v[a];
      const int id = sh.cand_i[a];
      int r = 0;
      for (int j = 0; j < n && r < k; ++j) r += before(sh.cand_v[j], sh.cand_i[j], v, id) ? 1 : 0;
      if (r < k) {
        sh.top_v[r] = v;
        sh.top_i[r] = id;
      }
    }
    __syncthreads();
    return;
  }
  float last_v = INFINITY;
  int last_i = -1;
  for (int r = 0; r < k; ++r) {  // the best element behind the last one chosen
    float bv = -INFINITY;
    int bi = 0x7fffffff;
    for_each<DT>(row, sl, [&](int64_t i, float x) {
      x = sort_key(x);
      if (before(last_v, last_i, x, (int)i) && before(x, (int)i, bv, bi)) {
        bv = x;
        bi = (int)i;
      }
    });
    for (int o = 16; o > 0; o >>= 1) {
      const float v2 = __shfl_xor_sync(0xffffffffu, bv, o);
      const int i2 = __shfl_xor_sync(0xffffffffu, bi, o);
      if (before(v2, i2, bv, bi)) {
        bv = v2;
        bi = i2;
      }
    }
    if ((tid & 31) == 0) {
      sh.red_v[tid >> 5] = bv;
      sh.red_i[tid >> 5] = bi;
    }
    __syncthreads();
    bv = sh.red_v[0];
    bi = sh.red_i[0];
    for (int j = 1; j < kWarps; ++j)
      if (before(sh.red_v[j], sh.red_i[j], bv, bi)) {
        bv = sh.red_v[j];
        bi = sh.red_i[j];
      }
    __syncthreads();
    if (tid == 0) {
      sh.top_v[r] = bv;
      sh.top_i[r] = bi;
    }
    last_v = bv;
    last_i = bi;
  }
  __syncthreads();
}

struct FwdArgs {
  const char *logits;
  int64_t row_bytes, V;
  const int64_t *tokens;
  int64_t ignore_index;
  float c;  // log2(e) / temperature
  float *logprob, *entropy, *top_logprob;
  double *lse;
  int64_t *top_id;
  int k;
};

template <int DT, bool CLUSTER, bool TOP>
__global__ void __launch_bounds__(kBlock, TOP ? 4 : 6) logprobs_fwd_kernel(const FwdArgs a) {
  __shared__ Shared sh;
  const int tid = threadIdx.x;
  int rank = 0, parts = 1;
  if (CLUSTER) {
    rank = (int)cg::this_cluster().block_rank();
    parts = (int)cg::this_cluster().num_blocks();
  }
  const int64_t r = blockIdx.x / parts;
  const char *row = a.logits + r * a.row_bytes;
  const Slice sl = slice_of<DT>(row, a.V, rank, parts);
  uint4 keep[kKeep];
  const bool kept = TOP && sl.nvec <= kKeep * kBlock;
  Stat t = sweep<DT>(row, sl, a.c, keep, kept);
  if (TOP) {
    local_top<DT>(row, sl, a.c, t.m, a.k, sh, keep, kept);
  }
  for (int o = 16; o > 0; o >>= 1) {
    const Stat u{__shfl_xor_sync(0xffffffffu, t.m, o), __shfl_xor_sync(0xffffffffu, t.s, o),
                 __shfl_xor_sync(0xffffffffu, t.w, o)};
    t = merge(t, u);
  }
  if ((tid & 31) == 0) sh.part[tid >> 5] = t;
  __syncthreads();
  t = sh.part[tid & (kWarps - 1)];  // the warps' triples, merged by every warp for itself
  for (int o = kWarps / 2; o > 0; o >>= 1) {
    const Stat u{__shfl_xor_sync(0xffffffffu, t.m, o), __shfl_xor_sync(0xffffffffu, t.s, o),
                 __shfl_xor_sync(0xffffffffu, t.w, o)};
    t = merge(t, u);
  }
  if (CLUSTER) {
    cg::cluster_group cl = cg::this_cluster();
    if (tid == 0) sh.total = t;
    cl.sync();
    if (rank == 0)
      for (int p = 1; p < parts; ++p) t = merge(t, *cl.map_shared_rank(&sh.total, p));
  }
  if (rank == 0) {
    const float l2 = log2f(t.s);
    const bool empty = t.m <= a.c * kStart && t.s == t.s;  // only masked logits in the row
    // masked logits have probability 0 at any temperature; the row's NaN comes first
    auto log_p = [&](float x) {
      return empty || (x < kStart && l2 == l2) ? -INFINITY : (fmaf(x, a.c, -t.m) - l2) * kLn2;
    };
    if (tid == 0) {
      const int64_t tok = a.tokens[r];
      float lp;
      if (tok == a.ignore_index)
        lp = 0.f;
      else if (tok < 0 || tok >= a.V)
        lp = NAN;
      else
        lp = log_p(Elem<DT>::load(row, tok));
      a.logprob[r] = lp;
      a.entropy[r] = empty ? 0.f : (l2 - t.w / t.s) * kLn2;
      a.lse[r] = empty ? -INFINITY : ((double)t.m + (double)l2) * kLn2D;
    }
    if (TOP) {
      // candidates: the CTAs' ordered lists, at most 8 x kTopMax = kBlock of them
      float v = -INFINITY;
      int id = 0x7fffffff;
      const int n = parts * a.k;
      if (tid < n) {
        const Shared *src = &sh;
        if (CLUSTER) src = cg::this_cluster().map_shared_rank(&sh, tid / a.k);
        v = src->top_v[tid % a.k];
        id = src->top_i[tid % a.k];
      }
      sh.cand_v[tid] = v;
      sh.cand_i[tid] = id;
      __syncthreads();
      if (tid < n) {
        int pos = 0;
        for (int j = 0; j < n; ++j) pos += before(sh.cand_v[j], sh.cand_i[j], v, id) ? 1 : 0;
        if (pos < a.k && id != 0x7fffffff) {
          a.top_logprob[r * a.k + pos] = log_p(v);
          a.top_id[r * a.k + pos] = id;
        }
      }
    }
  }
  if (CLUSTER) cg::this_cluster().sync();  // no CTA leaves while rank 0 reads its shared memory
}

struct BwdArgs {
  const char *logits;
  int64_t row_bytes, V;
  const int64_t *tokens;
  int64_t ignore_index;
  float c, inv_t;
  const float *entropy, *dlogprob, *dentropy;
  const double *lse;
  char *dlogits;  // [N, V] contiguous
};

template <int DT>
__global__ void __launch_bounds__(kBlock) logprobs_bwd_kernel(const BwdArgs g) {
  using E = Elem<DT>;
  const int64_t r = blockIdx.x;
  const char *row = g.logits + r * g.row_bytes;
  char *out = g.dlogits + r * g.V * E::kBytes;
  const int64_t tok = g.tokens[r];
  const bool counted = g.dlogprob != nullptr && tok != g.ignore_index;
  // lse in two fp32 terms: p's error is that of the exponent, and one term is off by 2^-24 of lse, which
  // over a low temperature or with a common offset of the logits is far more than the exponents that count
  const double lse = g.lse[r] * kLog2eD;
  const bool empty = lse == -INFINITY;
  const float l2 = empty ? 0.f : (float)lse, l2_low = empty ? 0.f : (float)(lse - (double)l2);
  // a token outside [0, V): its log probability is NaN, and so is the row's gradient through it
  const float a = !counted || empty ? 0.f : (tok < 0 || tok >= g.V) ? NAN : g.dlogprob[r] * g.inv_t;
  const float b = g.dentropy != nullptr && !empty ? g.dentropy[r] * g.inv_t : 0.f, H = g.entropy[r];
  const float base = -a - b * H, slope = -b * kLn2;
  const float low = (l2 + kFloor) / g.c;  // p is 0 from here down, where slope * d might overflow
  auto grad = [&](int64_t i, float x) {
    const float d = fmaf(floor1(x, low), g.c, -l2) - l2_low, p = ex2(d);
    float v = p * fmaf(slope, d, base);
    if (i == tok) v += a;
    return v;  // of an empty row: p = 0 everywhere, a = b = 0
  };
  const bool same = ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(out)) & 15u) == 0;
  if (!same) {
    for (int64_t i = threadIdx.x + (int64_t)blockIdx.y * kBlock; i < g.V; i += (int64_t)kBlock * gridDim.y)
      E::store(out, i, grad(i, E::load(row, i)));
    return;
  }
  const Slice sl = slice_of<DT>(row, g.V, blockIdx.y, gridDim.y);
  const uint4 *v4 = reinterpret_cast<const uint4 *>(row + sl.body * E::kBytes);
  uint4 *o4 = reinterpret_cast<uint4 *>(out + sl.body * E::kBytes);
  for (int64_t i = threadIdx.x; i < sl.nvec; i += kBlock) {
    float f[E::kVec];
    E::unpack(__ldg(v4 + i), f);
#pragma unroll
    for (int k = 0; k < E::kVec; ++k) f[k] = grad(sl.body + i * E::kVec + k, f[k]);
    o4[i] = E::pack(f);
  }
  for (int64_t i = sl.lo + threadIdx.x; i < sl.body; i += kBlock) E::store(out, i, grad(i, E::load(row, i)));
  for (int64_t i = sl.tail + threadIdx.x; i < sl.hi; i += kBlock) E::store(out, i, grad(i, E::load(row, i)));
}

int sm_count() {
  int dev = 0, n = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n > 0 ? n : 1;
}

// CTAs that share a row: enough to give every SM two, each with at least 2048 elements, up to
// the portable cluster size.
int parts_of(int64_t N, int64_t V) {
  const int64_t want = 2 * (int64_t)sm_count();
  int p = 1;
  while (p < 8 && N * p * 2 <= want && V / (p * 2) >= 2048) p *= 2;
  return p;
}

template <int DT, bool TOP>
cudaError_t launch_fwd_top(const FwdArgs &a, int64_t N, cudaStream_t st) {
  const int parts = parts_of(N, a.V);
  if (parts == 1) {
    logprobs_fwd_kernel<DT, false, TOP><<<(unsigned)N, kBlock, 0, st>>>(a);
    return cudaGetLastError();
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(N * parts));
  cfg.blockDim = dim3(kBlock);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = parts;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, logprobs_fwd_kernel<DT, true, TOP>, a);
  return e != cudaSuccess ? e : cudaGetLastError();
}

template <int DT>
cudaError_t launch_fwd(const FwdArgs &a, int64_t N, cudaStream_t st) {
  return a.k > 0 ? launch_fwd_top<DT, true>(a, N, st) : launch_fwd_top<DT, false>(a, N, st);
}

template <int DT>
cudaError_t launch_bwd(const BwdArgs &a, int64_t N, cudaStream_t st) {
  const int64_t want = 4 * (int64_t)sm_count();
  int64_t py = (want + N - 1) / N;
  const int64_t most = (a.V + 8191) / 8192;
  if (py > most) py = most;
  if (py < 1) py = 1;
  logprobs_bwd_kernel<DT><<<dim3((unsigned)N, (unsigned)py), kBlock, 0, st>>>(a);
  return cudaGetLastError();
}

int check(int64_t N, int64_t V, int64_t stride, float temperature, int32_t dtype) {
  if (N < 0 || V <= 0 || N > 0x7fffffff / 8 || V > 0x7ffffffe || (N > 1 && stride < V)) return KDA_ERR_BAD_SHAPE;
  if (!(temperature >= 1e-6f) || temperature > 1e6f) return KDA_ERR_UNSUPPORTED;  // c * kMask is finite
  if (dtype != kBF16 && dtype != kF16 && dtype != kF32) return KDA_ERR_UNSUPPORTED;
  return KDA_OK;
}

bool element_aligned(const void *p, int32_t dtype) {
  return (reinterpret_cast<uintptr_t>(p) & (dtype == kF32 ? 3u : 1u)) == 0;
}

}  // namespace

extern "C" {

int st_token_logprobs_fwd(const void *logits, int64_t row_stride, const int64_t *tokens, float *logprob, float *entropy,
                          double *lse, float *top_logprob, int64_t *top_id, int32_t top_k, int64_t N, int64_t V,
                          float temperature, int64_t ignore_index, int32_t dtype, kda_stream_t stream) {
  int rc = check(N, V, row_stride, temperature, dtype);
  if (rc != KDA_OK) return rc;
  if (top_k < 0 || top_k > V) return KDA_ERR_BAD_SHAPE;
  if (top_k > kTopMax) return KDA_ERR_UNSUPPORTED;
  if (N == 0) return KDA_OK;
  if (!logits || !tokens || !logprob || !entropy || !lse || (top_k > 0 && (!top_logprob || !top_id)))
    return KDA_ERR_NULL_ARGUMENT;
  if (!element_aligned(logits, dtype)) return KDA_ERR_BAD_LAYOUT;
  FwdArgs a{};
  a.logits = static_cast<const char *>(logits);
  a.row_bytes = row_stride * (dtype == kF32 ? 4 : 2);
  a.V = V;
  a.tokens = tokens;
  a.ignore_index = ignore_index;
  a.c = kLog2e / temperature;
  a.logprob = logprob;
  a.entropy = entropy;
  a.lse = lse;
  a.top_logprob = top_logprob;
  a.top_id = top_id;
  a.k = top_k;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == kBF16  ? launch_fwd<kBF16>(a, N, st)
                        : dtype == kF16 ? launch_fwd<kF16>(a, N, st)
                                        : launch_fwd<kF32>(a, N, st);
  kda::count_launches(1);
  return e == cudaSuccess ? KDA_OK : KDA_ERR_CUDA;
}

int st_token_logprobs_bwd(const void *logits, int64_t row_stride, const int64_t *tokens, const float *entropy,
                          const double *lse, const float *dlogprob, const float *dentropy, void *dlogits, int64_t N,
                          int64_t V, float temperature, int64_t ignore_index, int32_t dtype, kda_stream_t stream) {
  int rc = check(N, V, row_stride, temperature, dtype);
  if (rc != KDA_OK) return rc;
  if (N == 0) return KDA_OK;
  if (!logits || !tokens || !entropy || !lse || !dlogits) return KDA_ERR_NULL_ARGUMENT;
  if (!element_aligned(logits, dtype) || !element_aligned(dlogits, dtype)) return KDA_ERR_BAD_LAYOUT;
  BwdArgs a{};
  a.logits = static_cast<const char *>(logits);
  a.row_bytes = row_stride * (dtype == kF32 ? 4 : 2);
  a.V = V;
  a.tokens = tokens;
  a.ignore_index = ignore_index;
  a.inv_t = 1.f / temperature;
  a.c = kLog2e / temperature;
  a.entropy = entropy;
  a.lse = lse;
  a.dlogprob = dlogprob;
  a.dentropy = dentropy;
  a.dlogits = static_cast<char *>(dlogits);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == kBF16  ? launch_bwd<kBF16>(a, N, st)
                        : dtype == kF16 ? launch_bwd<kF16>(a, N, st)
                                        : launch_bwd<kF32>(a, N, st);
  kda::count_launches(1);
  return e == cudaSuccess ? KDA_OK : KDA_ERR_CUDA;
}

}  // extern "C"
