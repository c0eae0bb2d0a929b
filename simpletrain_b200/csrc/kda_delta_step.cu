// The gated delta rule for one new token per row, over a pool of fp32 states
// updated in place (C ABI in include/kda_sm100.h).
//
// Mathematics, per (row, head), S [D, D] with rows = key channels:
//   p = S^T k,  r = S^T q        (one read of S for both)
//   u = beta (v - a p),          a = exp(g)
//   o = scale (a r + (k . q) u)  (= scale S_new^T q, without a second read)
//   S <- a S + k u^T
// All in fp32; o is rounded once.
//
// Bound: HBM, 8 D^2 bytes a (row, head).  The columns of S are independent given
// k and q, so a CTA takes a slice of 32 columns (128-byte rows of S): 128 threads
// hold the slice in registers, 8 column quads x 16 groups of D/16 rows, with all
// their loads in flight at once, and the column sums meet through shuffles and
// shared memory.  Measured: 256 rows of 28 heads of 128, 947 MB, in 160 us: 5.9 TB/s, 0.92 of
// a copy's rate; one row of 8 heads of 64 takes 2.7 us, a launch and two dependent loads.
//
// Rows that name the same state are applied one after the other, in row order, by
// the CTA of the first of them: the result does not depend on the launch.  For that each CTA looks through all
// N indices, under its state's loads: with 24 heads of 128 it costs 4% at 256 rows, 8% at 1024, 42% at
// 4096 and 74% at 8192 (6.6 against 3.8 ms); rows that all name one state take 1.4 ms at 1024 and 24 ms at 8192.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/kda_sm100.h"
#include "kda_internal.h"
#include "tc_common.cuh"

namespace {

using kda::tc::pack2;
using kda::tc::unpack2;

constexpr int kBlock = 128;
constexpr int kCols = 32;

__device__ __forceinline__ float load_gate(const void *p, int64_t i, int dtype) {
  if (dtype == KDA_DTYPE_F32) return static_cast<const float *>(p)[i];
  return unpack2((uint32_t) static_cast<const uint16_t *>(p)[i], dtype == KDA_DTYPE_BF16).x;
}

template <int D>
__global__ void __launch_bounds__(kBlock) delta_step_kernel(const kda_delta_step_params a) {
  constexpr int R = D / 16;  // rows of S a thread
  __shared__ float4 sm_p[4][8], sm_r[4][8];
  __shared__ float sm_kq[4];
  __shared__ int sm_next;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cq = tid & 7, rg = tid >> 3;
  const int slices = D / kCols;
  const int sl = blockIdx.x % slices, h = (blockIdx.x / slices) % a.H;
  int64_t n = blockIdx.x / slices / a.H;
  const int col = sl * kCols + 4 * cq;
  const bool bf = a.dtype == KDA_DTYPE_BF16;
  int64_t slot = n, next = a.N;
  auto store_o = [&](int64_t row, float4 o) {
    uint2 w = make_uint2(pack2(o.x, o.y, bf), pack2(o.z, o.w, bf));
    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.o) + row * a.o_stride_n + h * a.o_stride_h + col) = w;
  };
  auto slot_of = [&](int64_t m) {
    return a.slots_int64 ? static_cast<const int64_t *>(a.slots)[m] : (int64_t) static_cast<const int32_t *>(a.slots)[m];
  };
  const int hk = h / (a.H / a.Hk);
  // a row's inputs; they do not depend on its state, so their latency is the index's and the state's too
  struct Row {
    uint32_t k[R / 2], q[R / 2];
    uint2 v;
    float alpha, beta;
  };
  auto load_row = [&](int64_t m) {
    Row r;
    const uint16_t *kp = static_cast<const uint16_t *>(a.k) + m * a.k_stride_n + hk * a.k_stride_h + rg * R;
    const uint16_t *qp = static_cast<const uint16_t *>(a.q) + m * a.q_stride_n + hk * a.q_stride_h + rg * R;
    if (R == 8) {
      *reinterpret_cast<uint4 *>(r.k) = *reinterpret_cast<const uint4 *>(kp);
      *reinterpret_cast<uint4 *>(r.q) = *reinterpret_cast<const uint4 *>(qp);
    } else {
      *reinterpret_cast<uint2 *>(r.k) = *reinterpret_cast<const uint2 *>(kp);
      *reinterpret_cast<uint2 *>(r.q) = *reinterpret_cast<const uint2 *>(qp);
    }
    r.v = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(a.v) + m * a.v_stride_n + h * a.v_stride_h + col);
    r.alpha = load_gate(a.g, m * a.g_stride_n + h * a.g_stride_h, a.g_dtype);
    r.beta = load_gate(a.beta, m * a.beta_stride_n + h * a.beta_stride_h, a.beta_dtype);
    return r;
  };
  if (a.slots != nullptr) slot = slot_of(n);
  Row in = load_row(n);
  if (a.slots != nullptr && (slot < 0 || slot >= a.num_states)) {  // a padded row (or an index that names no state)
    if (slot >= 0 && a.status != nullptr && tid == 0) atomicOr(a.status, KDA_ERR_DEVICE_INDEX);
    if (rg == 0) store_o(n, make_float4(0.f, 0.f, 0.f, 0.f));
    return;
  }
  float *S = a.state + slot * a.state_stride_n + h * a.state_stride_h + (int64_t)(rg * R) * D + col;
  float4 s[R];
#pragma unroll
  for (int i = 0; i < R; ++i) s[i] = *reinterpret_cast<const float4 *>(S + i * D);
  if (a.slots != nullptr) {  // under the state's loads: which other rows name this state?
    if (tid == 0) sm_next = a.N;
    __syncthreads();
    int dup = 0;
    for (int64_t m = tid; m < a.N; m += kBlock)
      if (m != n && slot_of(m) == slot) {
        if (m < n)
          dup = 1;
        else
          atomicMin(&sm_next, (int)m);
      }
    if (__syncthreads_or(dup)) return;  // an earlier row's CTA applies this row
    next = sm_next;
  }
  while (true) {
    float k[R], q[R];
#pragma unroll
    for (int i = 0; i < R / 2; ++i) {
      const float2 x = unpack2(in.k[i], bf), y = unpack2(in.q[i], bf);
      k[2 * i] = x.x;
      k[2 * i + 1] = x.y;
      q[2 * i] = y.x;
      q[2 * i + 1] = y.y;
    }
    const uint2 vw = in.v;
    const float alpha = expf(in.alpha), beta = in.beta;
    float4 p = make_float4(0.f, 0.f, 0.f, 0.f), r = p;
    float kq = 0.f;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      p.x = fmaf(s[i].x, k[i], p.x);
      p.y = fmaf(s[i].y, k[i], p.y);
      p.z = fmaf(s[i].z, k[i], p.z);
      p.w = fmaf(s[i].w, k[i], p.w);
      r.x = fmaf(s[i].x, q[i], r.x);
      r.y = fmaf(s[i].y, q[i], r.y);
      r.z = fmaf(s[i].z, q[i], r.z);
      r.w = fmaf(s[i].w, q[i], r.w);
      kq = fmaf(k[i], q[i], kq);
    }
#pragma unroll
    for (int o = 8; o < 32; o <<= 1) {
      p.x += __shfl_xor_sync(0xffffffffu, p.x, o);
      p.y += __shfl_xor_sync(0xffffffffu, p.y, o);
      p.z += __shfl_xor_sync(0xffffffffu, p.z, o);
      p.w += __shfl_xor_sync(0xffffffffu, p.w, o);
      r.x += __shfl_xor_sync(0xffffffffu, r.x, o);
      r.y += __shfl_xor_sync(0xffffffffu, r.y, o);
      r.z += __shfl_xor_sync(0xffffffffu, r.z, o);
      r.w += __shfl_xor_sync(0xffffffffu, r.w, o);
      kq += __shfl_xor_sync(0xffffffffu, kq, o);
    }
    if (lane < 8) {
      sm_p[warp][cq] = p;
      sm_r[warp][cq] = r;
      if (lane == 0) sm_kq[warp] = kq;
    }
    __syncthreads();
    p = sm_p[0][cq];
    r = sm_r[0][cq];
    kq = sm_kq[0];
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      const float4 x = sm_p[w][cq], y = sm_r[w][cq];
      p.x += x.x; p.y += x.y; p.z += x.z; p.w += x.w;
      r.x += y.x; r.y += y.y; r.z += y.z; r.w += y.w;
      kq += sm_kq[w];
    }
    const float2 v01 = unpack2(vw.x, bf), v23 = unpack2(vw.y, bf);
    const float4 u = make_float4(beta * (v01.x - alpha * p.x), beta * (v01.y - alpha * p.y),
                                 beta * (v23.x - alpha * p.z), beta * (v23.y - alpha * p.w));
    if (rg == 0)
      store_o(n, make_float4(a.scale * fmaf(kq, u.x, alpha * r.x), a.scale * fmaf(kq, u.y, alpha * r.y),
                             a.scale * fmaf(kq, u.z, alpha * r.z), a.scale * fmaf(kq, u.w, alpha * r.w)));
#pragma unroll
    for (int i = 0; i < R; ++i) {
      s[i].x = fmaf(k[i], u.x, alpha * s[i].x);
      s[i].y = fmaf(k[i], u.y, alpha * s[i].y);
      s[i].z = fmaf(k[i], u.z, alpha * s[i].z);
      s[i].w = fmaf(k[i], u.w, alpha * s[i].w);
    }
    if (next >= a.N) break;
    n = next;  // the next row of the same state
    in = load_row(n);
    __syncthreads();
    if (tid == 0) sm_next = a.N;
    __syncthreads();
    for (int64_t m = n + 1 + tid; m < a.N; m += kBlock)
      if (slot_of(m) == slot) atomicMin(&sm_next, (int)m);
    __syncthreads();
    next = sm_next;
  }
#pragma unroll
  for (int i = 0; i < R; ++i) *reinterpret_cast<float4 *>(S + i * D) = s[i];
}

bool gate_ok(int32_t d) { return d == KDA_DTYPE_BF16 || d == KDA_DTYPE_F16 || d == KDA_DTYPE_F32; }

}  // namespace

extern "C" int kda_delta_step_sm100(const kda_delta_step_params *p, kda_stream_t stream) {
  if (p == nullptr) return KDA_ERR_NULL_ARGUMENT;
  const kda_delta_step_params &a = *p;
  if (a.N < 0 || a.H < 0 || a.Hk < 0 || a.num_states < 0) return KDA_ERR_BAD_SHAPE;
  if (a.D != 64 && a.D != 128) return KDA_ERR_UNSUPPORTED;
  if (a.dtype != KDA_DTYPE_BF16 && a.dtype != KDA_DTYPE_F16) return KDA_ERR_UNSUPPORTED;
  if (!gate_ok(a.g_dtype) || !gate_ok(a.beta_dtype)) return KDA_ERR_UNSUPPORTED;
  if (a.N == 0 || a.H == 0) return KDA_OK;
  if (a.Hk == 0 || a.H % a.Hk) return KDA_ERR_BAD_SHAPE;
  if (a.slots == nullptr && a.N > a.num_states) return KDA_ERR_BAD_SHAPE;
  const int64_t ctas = (int64_t)a.N * a.H * (a.D / kCols);
  if (ctas > 0x7fffffff) return KDA_ERR_BAD_SHAPE;
  if (!a.q || !a.k || !a.v || !a.o || !a.g || !a.beta || (!a.state && a.num_states > 0)) return KDA_ERR_NULL_ARGUMENT;
  const uintptr_t b16[] = {(uintptr_t)a.q, (uintptr_t)a.k, (uintptr_t)a.v, (uintptr_t)a.o, (uintptr_t)a.state};
  for (uintptr_t x : b16)
    if (x & 15u) return KDA_ERR_BAD_LAYOUT;
  const int64_t st[] = {a.q_stride_n, a.q_stride_h, a.k_stride_n, a.k_stride_h,
                        a.v_stride_n, a.v_stride_h, a.o_stride_n, a.o_stride_h};
  for (int64_t x : st)
    if (x % 8) return KDA_ERR_BAD_LAYOUT;
  if (a.state_stride_n % 4 || a.state_stride_h % 4) return KDA_ERR_BAD_LAYOUT;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (a.D == 64)
    delta_step_kernel<64><<<(unsigned)ctas, kBlock, 0, s>>>(a);
  else
    delta_step_kernel<128><<<(unsigned)ctas, kBlock, 0, s>>>(a);
  kda::count_launches(1);
  return cudaGetLastError() == cudaSuccess ? KDA_OK : KDA_ERR_CUDA;
}
