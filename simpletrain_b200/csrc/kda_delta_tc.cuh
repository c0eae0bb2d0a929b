// Pieces shared by the gated delta rule's kernels: arguments, sequence and chunk
// bookkeeping, tile loads, the two-term operand split, and MMA issue.
//
// Two-term operands.  A value x that is not an input is handed to the tensor cores as
// hi + lo, hi = round16(x), lo = round16(x - hi): 16 bits of mantissa in bf16, 22 in
// fp16 (whose exponents need the units below for that), against 8 and 11 in one term.  A product of two such values is issued as
// hi*hi + hi*lo + lo*hi into one fp32 accumulator.  With single terms the state,
// which feeds on itself chunk after chunk, was 2.5e-3 from the 64-bit recurrence;
// with two it is 4e-6, and the tensor pipe is not what bounds these kernels.  (Where keys repeat, an error
// of an operand is multiplied by the row sums of |T|, up to 1 + beta / (1 - |1 - beta|): 1e-5 at beta = 1, 1e-4 at 1.9.)
//
// Units (fp16 only).  fp16 ends at 65504, and its two terms have their 22 bits from about 2^-3 up: a
// gradient of 1e-5, as a loss's mean gives, left ds0 7% off, and a state past 65504 became infinite.  The
// recurrence is linear in (S, V) and its reverse in (dS, dO), so within a chunk everything that is
// split is carried times a power of two, chosen from the largest elements of both so that they lie at
// 2^6 to 2^7: 2^9 of room above for what a chunk's products make of them, 2^9 below before a
// bit is lost.  Products and sums are scaled back in fp32, which is exact.  Results in fp32 are 6e-7 to 1e-6 from the
// recurrence whatever the sizes (test inputs of 1e-5 to 1e5).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "../../include/kda_sm100.h"
#include "kda_internal.h"
#include "tc_common.cuh"

namespace kda {
namespace delta {

using namespace kda::tc;

constexpr int kChunk = 64;
constexpr int kImgT = 32768;  // T / PT image of a (chunk, head): [128 x 64] hi, then lo
constexpr double kLog2e = 1.4426950408889634;
constexpr float kMinGate = -110.f;  // exp() is 0 in fp32 from about -104 on

// Workspace regions (device pointers) of one call.
struct Work {
  int *queue;      // [2 scans][2 + ranges]: ticket, then a flag a range whose entry state is published; cleared by the preparation
  float *slots;    // [scan][ranges + 1][D][D] states at the ranges' boundaries
  float2 *cuts;    // fp16: [scan][ranges + 1][8] a warp of the chain each: how large a slot's state is at most, in two parts
  int *bound;      // [nseq + 1] sequence offsets, clamped into order and range (packed sequences only)
  int *first;      // [nseq + 1] first chunk of each sequence
  float *gam;      // [chunk][H][2][64] running sums of the log decay inside the chunk, in units of log 2 and in two
                   // terms: their differences decide the factors, and after a few strong decays (-110 each) one
                   // fp32 term is 1e-4 from the sum (the state was 2e-4 from the recurrence's)
  float *beta;     // [chunk][H][64]
  float *unit;     // fp16: [chunk][H][kUnits], see below
  char *T;         // [chunk][H] images of T over P T
  char *S, *dS;    // [chunk][H] images of the state before / the state gradient after the chunk, transposed: hi,
                   // then lo, each D / 8 runs of [D value rows x 8 key channels]
  char *U;         // [chunk][H] images of the chunk's u rows, transposed: hi, then lo, each 8 runs of [D value rows x 8 tokens]
  char *dX;        // [chunk][H][D / 64] images of the gradient of X: [64 tokens x 64] hi, then lo
};

// Of a (chunk, head), from the preparation: 1 / unit of P T, and the largest of 1 and |beta|, of |scale| and |P|,
// of |k_t|; from the scans: 1 / unit of the S and U images, and of the dS and dX images.
enum { kUnitP = 0, kSizeB = 1, kSizeP = 2, kSizeK = 3, kUnitF = 4, kUnitR = 5, kUnits = 8 };

struct Args {
  kda_delta_params p;
  Work w;
  int nseq;       // sequences (batch rows, or those of cu_seqlens)
  int per_seq;    // chunks of a batch row (without cu_seqlens)
  int max_chunks; // upper bound of the chunks over all sequences
  int ranges;     // CTAs of a scan
  int sms;        // of the device
};

struct Seq {
  int64_t b, t0;  // batch row and first token
  int len, chunk0;
};

__device__ __forceinline__ Seq get_seq(const Args &a, int n) {
  if (a.p.cu_seqlens == nullptr) return {n, 0, a.p.T, n * a.per_seq};
  const int lo = a.w.bound[n];
  return {0, lo, a.w.bound[n + 1] - lo, a.w.first[n]};
}

// Chunk u as (sequence, first token in it, rows); false past the last chunk.
__device__ __forceinline__ bool get_chunk(const Args &a, int u, int64_t *b, int64_t *t, int *rows) {
  if (a.p.cu_seqlens == nullptr) {
    const int n = u / a.per_seq, c = u - n * a.per_seq;
    *b = n;
    *t = (int64_t)c * kChunk;
    *rows = min(kChunk, a.p.T - c * kChunk);
    return true;
  }
  if (u >= a.w.first[a.nseq]) return false;
  int lo = 0, hi = a.nseq;  // first[lo] <= u < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.w.first[mid] <= u) lo = mid; else hi = mid;
  }
  const int c = u - a.w.first[lo], s0 = a.w.bound[lo];
  *b = 0;
  *t = (int64_t)s0 + (int64_t)c * kChunk;
  *rows = min(kChunk, a.w.bound[lo + 1] - s0 - c * kChunk);
  return true;
}

__device__ __forceinline__ float ex2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// e^{gamma_i - gamma_j} from two-term gammas
__device__ __forceinline__ float decay(float hi_i, float lo_i, float hi_j, float lo_j) { return ex2f((hi_i - hi_j) + (lo_i - lo_j)); }

__device__ __forceinline__ float load_gate(const void *p, int64_t i, int dtype) {
  if (dtype == KDA_DTYPE_F32) return static_cast<const float *>(p)[i];
  return unpack2((uint32_t) static_cast<const uint16_t *>(p)[i], dtype == KDA_DTYPE_BF16).x;
}
__device__ __forceinline__ void store_gate(void *p, int64_t i, int dtype, float v) {
  if (dtype == KDA_DTYPE_F32)
    static_cast<float *>(p)[i] = v;
  else
    static_cast<uint16_t *>(p)[i] = (uint16_t)(pack2(v, 0.f, dtype == KDA_DTYPE_BF16) & 0xffffu);
}

// The unit of numbers up to m (the bits of a value >= 0) and its inverse.  NaN and infinity: 1, they pass through.
__device__ __forceinline__ float unit_of(uint32_t m, float *inverse) {
  int e = (int)(m >> 23) - 127;
  e = m >= 0x7f800000u ? 6 : min(max(e, -60), 80);
  *inverse = __uint_as_float((uint32_t)(127 - 6 + e) << 23);
  return __uint_as_float((uint32_t)(127 + 6 - e) << 23);
}
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
// the larger one of both halves of eight fp16 values, as bits of |x|
__device__ __forceinline__ uint32_t half_size(const uint4 &v) {
  const uint32_t m = 0x7fff7fffu, x = __vmaxu2(__vmaxu2(v.x & m, v.y & m), __vmaxu2(v.z & m, v.w & m));
  return max(x & 0xffffu, x >> 16);
}

// ------------------------------------------------------------- tile loads --
// 16 bytes to shared memory, zeros where `live` is false (the source is not read then)
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// `rows` live rows (of 64) of a [T, D] view at `base` into rows [row0, row0 + 64) of D/64
// swizzled [128 x 64] blocks, by THREADS threads; rows past `rows` become zeros.
template <int D, int THREADS>
__device__ __forceinline__ void load_rows(uint32_t tile, int row0, const uint16_t *base, int64_t stride_t, int rows) {
  constexpr int P = D / 8;
#pragma unroll
  for (int i = 0; i < 64 * P / THREADS; ++i) {
    const int p = threadIdx.x + i * THREADS, r = p / P, c = p % P, tr = row0 + r;
    const bool live = r < rows;
    cp_async16(tile + (c >> 3) * 16384 + tr * 128 + (((c & 7) ^ (tr & 7)) << 4), base + (live ? r * stride_t : 0) + c * 8, live);
  }
}

// Announce bytes to an mbarrier's phase without arriving on it.
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// contiguous bytes global -> shared, counted on an mbarrier (sizes and addresses are multiples of 16)
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void bulk_store(void *dst, uint32_t src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(reinterpret_cast<uint64_t>(dst)),
               "r"(src), "r"(bytes)
               : "memory");
}

// ------------------------------------------------------------ hi/lo split --
// lo = round16(x - hi), the difference by a mixed-precision fma that takes hi as it is packed
template <bool BF>
__device__ __forceinline__ void split2(float a, float b, uint32_t &hi, uint32_t &lo) {
  hi = pack2(a, b, BF);
  float x, y;
  if (BF)
    asm("{\n\t.reg .b16 l, h, m;\n\tmov.b32 {l, h}, %2;\n\tmov.b16 m, 0xBF80;\n\t"
        "fma.rn.f32.bf16 %0, l, m, %3;\n\tfma.rn.f32.bf16 %1, h, m, %4;\n\t}"
        : "=f"(x), "=f"(y)
        : "r"(hi), "f"(a), "f"(b));
  else
    asm("{\n\t.reg .b16 l, h, m;\n\tmov.b32 {l, h}, %2;\n\tmov.b16 m, 0xBC00;\n\t"
        "fma.rn.f32.f16 %0, l, m, %3;\n\tfma.rn.f32.f16 %1, h, m, %4;\n\t}"
        : "=f"(x), "=f"(y)
        : "r"(hi), "f"(a), "f"(b));
  lo = pack2(x, y, BF);
}

// Eight consecutive columns (16-byte chunk c16) of row `row` of a swizzled tile, as hi and lo.
template <bool BF>
__device__ __forceinline__ void split8(const float *x, uint4 &hi, uint4 &lo) {
  split2<BF>(x[0], x[1], hi.x, lo.x);
  split2<BF>(x[2], x[3], hi.y, lo.y);
  split2<BF>(x[4], x[5], hi.z, lo.z);
  split2<BF>(x[6], x[7], hi.w, lo.w);
}
__device__ __forceinline__ uint32_t chunk_at(int row, int c16) {
  return (uint32_t)(row * 128 + (((c16 ^ row) & 7) << 4));
}
__device__ __forceinline__ void sts(uint32_t addr, const uint4 &v) { st_shared_v4(addr, v.x, v.y, v.z, v.w); }

// 16 columns (chunks c16 and c16 + 1) of a row into the hi and lo tiles
template <bool BF>
__device__ __forceinline__ void store_split16(uint32_t hi_tile, uint32_t lo_tile, int row, int c16, const float (&x)[16]) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint4 h, l;
    split8<BF>(x + 8 * c, h, l);
    const uint32_t at = chunk_at(row, c16 + c);
    sts(hi_tile + at, h);
    sts(lo_tile + at, l);
  }
}
template <bool BF>
__device__ __forceinline__ void unpack8(const uint4 &v, float *f) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = unpack2(w[i], BF);
    f[2 * i] = p.x;
    f[2 * i + 1] = p.y;
  }
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&x)[32]) {
  uint32_t r[32];
  tmem_ld_32x32b_x32(taddr, r);
#pragma unroll
  for (int i = 0; i < 32; ++i) x[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&x)[16]) {
  uint32_t r[16];
  tmem_ld_32x32b_x16(taddr, r);
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const float (&x)[16]) {
  uint32_t r[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(x[i]);
  tmem_st_32x32b_x16(taddr, r);
}
// -------------------------------------------------------------- MMA issue --
// Operand views of a swizzled tile: K-major (rows are M or N, 64-column blocks `block`
// bytes apart along K) or MN-major (rows are K, 64-column blocks `block` bytes apart
// along M or N).  Step ks covers K elements [16 ks, 16 ks + 16).  One thread issues all
// products, so a step costs it an add to the descriptor's address field, no more.
struct KMajor {
  uint64_t base;
  uint32_t block;
  __device__ __forceinline__ KMajor(uint32_t at, uint32_t block_) : base(sdesc_k(at)), block(block_ >> 4) {}
  __device__ __forceinline__ uint64_t desc(int ks) const { return base + (uint64_t)((ks >> 2) * block + (ks & 3) * 2); }
};
struct MNMajor {
  uint64_t base;
  __device__ __forceinline__ MNMajor(uint32_t at, uint32_t block_) : base(sdesc_mn(at, block_)) {}
  __device__ __forceinline__ uint64_t desc(int ks) const { return base + (uint64_t)(ks * 128); }
};
// MN-major without swizzle, the order in which the scans write their images: 16-byte runs of
// eight M or N elements, one K row after the other (`rows` rows a run of 8 elements).
struct MNPlain {
  uint64_t base;
  __device__ __forceinline__ MNPlain(uint32_t at, uint32_t rows)
      : base((uint64_t)((at >> 4) & 0x3FFFu) | (uint64_t)8 << 16 | (uint64_t)(rows & 0x3FFFu) << 32 | (uint64_t)1 << 46) {}
  __device__ __forceinline__ uint64_t desc(int ks) const { return base + (uint64_t)(ks * 16); }
};
template <int STEPS, typename A, typename B>
__device__ __forceinline__ void issue(uint32_t d, const A &a, const B &b, uint32_t idesc, bool accumulate) {
#pragma unroll
  for (int ks = 0; ks < STEPS; ++ks) mma_f16(d, a.desc(ks), b.desc(ks), idesc, (accumulate || ks > 0) ? 1u : 0u);
}

// One lane of a converged warp.  A branch on it tells the compiler that a single thread
// issues, and a product then costs 27 cycles to issue against 46 behind a branch on the
// lane number and 64 when every product is predicated (M = 128, N = 64, K = 16).
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}
// the thread that issues a CTA's products
__device__ __forceinline__ bool warp_leader() { return threadIdx.x < 32 && elect_one(); }
// first operand in tensor memory: rows = lanes, two consecutive K elements a column
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// products with steps [K0, K1) of B and of A (tensor memory, eight columns a step)
template <int K0, int K1, typename B>
__device__ __forceinline__ void issue_ts(uint32_t d, uint32_t a, const B &b, uint32_t idesc, bool accumulate) {
#pragma unroll
  for (int ks = K0; ks < K1; ++ks) mma_f16_ts(d, a + 8 * ks, b.desc(ks), idesc, (accumulate || ks > K0) ? 1u : 0u);
}
template <int K0, int K1, typename A, typename B>
__device__ __forceinline__ void issue_ss(uint32_t d, const A &a, const B &b, uint32_t idesc, bool accumulate) {
#pragma unroll
  for (int ks = K0; ks < K1; ++ks) mma_f16(d, a.desc(ks), b.desc(ks), idesc, (accumulate || ks > K0) ? 1u : 0u);
}

// --------------------------------------------------------- CTA scaffolding --
struct Ctl {
  uint64_t mma_bar, load_bar;
  uint32_t tmem;
  int abort;
};

// Barriers and tensor memory; returns the tensor-memory base.
__device__ __forceinline__ uint32_t cta_begin(Ctl &ctl, uint32_t cols) {
  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&ctl.mma_bar), 1);
    mbar_init(smem_u32(&ctl.load_bar), 1);
    mbar_fence_init();
    ctl.abort = 0;
  }
  if (threadIdx.x < 32) {
    tmem_alloc(smem_u32(&ctl.tmem), cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  return *reinterpret_cast<volatile uint32_t *>(&ctl.tmem);
}
__device__ __forceinline__ void cta_end(uint32_t tmem, uint32_t cols) {
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (threadIdx.x < 32) tmem_dealloc(tmem, cols);
}
// Writes of this thread to shared and tensor memory before the barrier are seen by the
// products issued after it.
__device__ __forceinline__ void publish() {
  fence_async_smem();
  tc_fence_before();
  __syncthreads();
}
__device__ __forceinline__ void wait_bar(uint64_t &bar, uint32_t &phase, Ctl &ctl, int32_t *status) {
  mbar_wait(smem_u32(&bar), phase, status, &ctl.abort);
  phase ^= 1;
  __syncwarp();
  tc_fence_after();
}

// Allow `kern` `smem` bytes of dynamic shared memory on the current device, once a device (`done`: a
// bit for each, kept by the caller).
template <typename K>
cudaError_t allow_smem(K kern, uint32_t smem, std::atomic<uint64_t> &done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

// launchers (kda_delta_scan.cu, kda_delta_grad.cu)
cudaError_t launch_plan(const Args &a, cudaStream_t st);
cudaError_t launch_prep(const Args &a, cudaStream_t st);
cudaError_t launch_scan(const Args &a, cudaStream_t st);           // outputs
cudaError_t launch_backward_scans(const Args &a, cudaStream_t st);  // states and u rows, then the reverse scan
cudaError_t launch_grad(const Args &a, cudaStream_t st);

}  // namespace delta
}  // namespace kda
