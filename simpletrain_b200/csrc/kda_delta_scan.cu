// The gated delta rule over chunks of 64 tokens: chunk preparation, the forward scan
// and the reverse (state gradient) scan.
//
// Mathematics, per (sequence, head) and chunk, gamma_i the running sum of the log decay
// inside the chunk, G = e^gamma, last = e^{gamma_63}:
//   A_ij = beta_i e^{gamma_i - gamma_j} k_i.k_j (i > j)     T = (I + A)^-1
//   P_ij = scale e^{gamma_i - gamma_j} q_i.k_j (i >= j)
//   X = beta (V - G K S)     U = T X     O = scale G Q S + (P T) X
//   S <- last S + K^T (e^{gamma_63 - gamma} U)
// and, for dS the gradient of the state after the chunk,
//   Z = e^{gamma_63 - gamma} K dS     dX = (P T)^T dO + T^T Z     dV = beta dX
//   dS <- last dS + K^T (-G beta dX) + Q^T (scale G dO)
// Every exponent is of a difference <= 0 for g <= 0, so no factor overflows.
//
// T and P T depend on one chunk alone: a first kernel forms them for all chunks at once,
// and the scans, which are sequential in the chunks, are left with three dependent
// products a chunk: with the state, with T (or its transpose), and the state update, which
// accumulates on the state in tensor memory.
#include "kda_delta_ranges.h"
#include "kda_delta_tc.cuh"
#include "tmap.h"

namespace kda {
namespace delta {
namespace {

// ------------------------------------------------------------ sequence plan --
// bound[i] = cu_seqlens[i] clamped into [0, T] and to no less than its predecessors;
// first[i] = chunks before sequence i.
__global__ void __launch_bounds__(1024) plan_kernel(const Args a) {
  pdl_launch_dependents();
  __shared__ int sm_max[32], sm_sum[32];
  __shared__ int carry_max, carry_sum;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = a.nseq;
  if (tid == 0) {
    carry_max = 0;
    carry_sum = 0;
  }
  __syncthreads();
  int bad = 0;
  for (int base = 0; base <= n; base += 1024) {
    const int i = base + tid;
    int64_t raw = 0;
    if (i <= n)
      raw = a.p.cu_int64 ? static_cast<const int64_t *>(a.p.cu_seqlens)[i] : static_cast<const int32_t *>(a.p.cu_seqlens)[i];
    int m = (int)(raw < 0 ? 0 : (raw > a.p.T ? a.p.T : raw));
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, m, o);
      if (lane >= o) m = max(m, y);
    }
    if (lane == 31) sm_max[warp] = m;
    __syncthreads();
    int before = carry_max;
    for (int w = 0; w < warp; ++w) before = max(before, sm_max[w]);
    m = max(m, before);
    // chunks of the sequence that ends at i (sequence i - 1)
    int prev = __shfl_up_sync(0xffffffffu, m, 1);
    if (lane == 0) prev = before;
    int c = (i >= 1 && i <= n) ? (m - prev + kChunk - 1) / kChunk : 0;
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, c, o);
      if (lane >= o) c += y;
    }
    if (lane == 31) sm_sum[warp] = c;
    __syncthreads();
    int sum = carry_sum;
    for (int w = 0; w < warp; ++w) sum += sm_sum[w];
    c += sum;
    if (i <= n) {
      a.w.bound[i] = m;
      a.w.first[i] = c;
      bad |= m != raw;
    }
    __syncthreads();
    if (tid == 1023) {
      carry_max = m;
      carry_sum = c;
    }
    __syncthreads();
  }
  if (bad && a.p.status != nullptr) atomicOr(a.p.status, KDA_ERR_DEVICE_INDEX);
}

// -------------------------------------------------------------- preparation --
constexpr int kLd = 68;  // row stride (floats) of the fp32 64 x 64 matrices: vectors of 8 rows in distinct banks

// Two rows and four columns of sign * L R, with n terms: eight sums a thread on six 16-byte
// loads every four terms (one row a thread spent its time on the loads).
template <int n>
__device__ __forceinline__ void block_product(const float *l, const float *r, float *out, float sign) {
  float4 s0 = make_float4(0.f, 0.f, 0.f, 0.f), s1 = s0;
  auto add = [](float4 &s, float f, const float4 &v) {
    s.x = fmaf(f, v.x, s.x);
    s.y = fmaf(f, v.y, s.y);
    s.z = fmaf(f, v.z, s.z);
    s.w = fmaf(f, v.w, s.w);
  };
#pragma unroll 4
  for (int m = 0; m < n; m += 4) {
    const float4 l0 = *reinterpret_cast<const float4 *>(l + m), l1 = *reinterpret_cast<const float4 *>(l + kLd + m);
    const float4 r0 = *reinterpret_cast<const float4 *>(r + m * kLd), r1 = *reinterpret_cast<const float4 *>(r + (m + 1) * kLd);
    const float4 r2 = *reinterpret_cast<const float4 *>(r + (m + 2) * kLd), r3 = *reinterpret_cast<const float4 *>(r + (m + 3) * kLd);
    add(s0, l0.x, r0);
    add(s1, l1.x, r0);
    add(s0, l0.y, r1);
    add(s1, l1.y, r1);
    add(s0, l0.z, r2);
    add(s1, l1.z, r2);
    add(s0, l0.w, r3);
    add(s1, l1.w, r3);
  }
  *reinterpret_cast<float4 *>(out) = make_float4(sign * s0.x, sign * s0.y, sign * s0.z, sign * s0.w);
  *reinterpret_cast<float4 *>(out + kLd) = make_float4(sign * s1.x, sign * s1.y, sign * s1.z, sign * s1.w);
}

// For each pair of diagonal n-blocks of the inverse, the block below them: -c B a, through the
// unused block of A above them.
template <int n>
__device__ __forceinline__ void inverse_level(float *As, float *Ti) {
  const int p = threadIdx.x / (n * n / 8), f = threadIdx.x % (n * n / 8), i = f / (n / 4) * 2, j = f % (n / 4) * 4, o = 2 * n * p;
  if (p < 32 / n) block_product<n>(As + (o + n + i) * kLd + o, Ti + o * kLd + o + j, As + (o + i) * kLd + o + n + j, 1.f);
  __syncthreads();
  if (p < 32 / n) block_product<n>(Ti + (o + n + i) * kLd + o + n, As + o * kLd + o + n + j, Ti + (o + n + i) * kLd + o + j, -1.f);
  __syncthreads();
}

// One CTA per (chunk, head): T and P T as two-term images, gamma and beta in fp32.
// The products are k.k, q.k and P T; (I + A)^-1 is by halves in fp32: four 16 x 16 blocks
// by substitution, a column a thread, then [A 0; B C]^-1 = [a 0; -c B a, c] twice.
// The q.k rows wait in tensor memory while the inverse is formed, so that the k and q tiles, the
// fp32 matrices and the two-term tiles can take turns in 34 KB, and four CTAs share an SM: a cell is a
// chain of short dependent steps, hidden by other CTAs only.
//
// Measured: 110 us for 16 x 2048 tokens, 10 heads of 128 (5120 cells, 64 KB of k, q and images each:
// 3.1 TB/s).  The shared-memory pipe sets that (77% of its cycles taken, the tensor pipe 13%): 128 threads a
// CTA and six CTAs an SM, persistent CTAs that load the next cell under this one, and half the loads
// in the inverse's upper level all came to the same time.  In fp16, with P's unit and the sizes, 117 us.
constexpr int kPrepThreads = 256;

template <int D, bool BF>
__global__ void __launch_bounds__(kPrepThreads, 4) prep_kernel(const Args a) {
  constexpr uint32_t KQ = 0, TT = 0;  // [T; P] hi, then lo, over the rest
  extern __shared__ __align__(1024) char smem[];
  __shared__ Ctl ctl;
  __shared__ __align__(16) float gam[2][64], bet[64];
  __shared__ uint32_t size[3];  // fp16: the largest |beta|, |P| and k_t.k_t, as bits
  int64_t b, t0;
  int rows;
  if (a.p.cu_seqlens != nullptr) pdl_wait();  // for the plan
  pdl_launch_dependents();
  if (blockIdx.x == 0 && blockIdx.y == 0)
    for (int i = threadIdx.x; i < 2 * (a.ranges + 2); i += kPrepThreads) a.w.queue[i] = 0;
  if (!get_chunk(a, blockIdx.x, &b, &t0, &rows)) return;
  const int h = blockIdx.y, hk = h / (a.p.H / a.p.Hk), tid = threadIdx.x;
  const int row = tid & 127, half = tid >> 7, r64 = row & 63;
  const uint32_t sb = smem_u32(smem), lane_base = (uint32_t)((tid >> 5) & 3) << 21;
  load_rows<D, kPrepThreads>(sb + KQ, 0, static_cast<const uint16_t *>(a.p.k.data) + b * a.p.k.stride_b + hk * a.p.k.stride_h + t0 * a.p.k.stride_t,
               a.p.k.stride_t, rows);
  load_rows<D, kPrepThreads>(sb + KQ, 64, static_cast<const uint16_t *>(a.p.q.data) + b * a.p.q.stride_b + hk * a.p.q.stride_h + t0 * a.p.q.stride_t,
               a.p.q.stride_t, rows);
  if (!BF && tid < 3) size[tid] = 0;
  const uint32_t tmem = cta_begin(ctl, 64);
  const size_t ch = (size_t)blockIdx.x * a.p.H + h;
  if (tid < 32) {
    // running sums in double, then in two fp32 terms
    double s[2];
    for (int j = 0; j < 2; ++j) {
      const int i = 2 * tid + j;
      const float gate = i < rows ? load_gate(a.p.g, b * a.p.g_stride_b + h * a.p.g_stride_h + (t0 + i) * a.p.g_stride_t, a.p.g_dtype) : 0.f;
      s[j] = gate < kMinGate ? kMinGate : gate;  // a NaN stays one
      bet[i] = i < rows ? load_gate(a.p.beta, b * a.p.beta_stride_b + h * a.p.beta_stride_h + (t0 + i) * a.p.beta_stride_t, a.p.beta_dtype) : 0.f;
      if constexpr (!BF) atomicMax(&size[0], abs_bits(bet[i]));
    }
    double c = s[0] + s[1];
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, c, o);
      if (tid >= o) c += y;
    }
    for (int j = 0; j < 2; ++j) {
      const double x = kLog2e * (j ? c : c - s[1]);
      const float hi = (float)x;
      gam[0][2 * tid + j] = hi;
      gam[1][2 * tid + j] = (float)(x - (double)hi);
    }
  }
  cp_async_wait();
  publish();
  uint32_t ph = 0;
  if (warp_leader()) {
    tc_fence_after();
    issue<D / 16>(tmem, KMajor{sb + KQ, 16384}, KMajor{sb + KQ, 16384}, idesc_f16(128, 64, BF, false, false), false);
    mma_commit(smem_u32(&ctl.mma_bar));
  }
  if (tid < 128) a.w.gam[ch * 128 + tid] = gam[tid >> 6][tid & 63];
  if (tid < 64) a.w.beta[ch * 64 + tid] = bet[tid];
  const float gh = gam[0][r64], gl = gam[1][r64];
  const float rowf = row < 64 ? bet[r64] : a.p.scale;
  wait_bar(ctl.mma_bar, ph, ctl, a.p.status);
  float *As = reinterpret_cast<float *>(smem + KQ);  // over the k and q tiles: their product is done
  float *Ti = As + 64 * kLd;
  const uint32_t taddr = tmem + lane_base + 32 * half;
  // 16 columns at a time of a row of A (rows of k) or P (rows of q)
  const int last = r64 - (row < 64 ? 1 : 0) - 32 * half;  // last column that counts
  uint32_t mp = 0;
#pragma unroll
  for (int c0 = 0; c0 < 32; c0 += 16) {
    float x[16];
    tmem_ld16(taddr + c0, x);
    if constexpr (!BF) {
      const int own = r64 - 32 * half - c0;  // k_t.k_t
      if (row < 64 && own >= 0 && own < 16) {
        float kk = 0.f;
#pragma unroll
        for (int j = 0; j < 16; ++j) kk = j == own ? x[j] : kk;
        atomicMax(&size[2], abs_bits(kk));
      }
    }
#pragma unroll
    for (int j = 0; j < 16; j += 4) {
      const float4 c = *reinterpret_cast<const float4 *>(gam[0] + 32 * half + c0 + j);
      const float4 l = *reinterpret_cast<const float4 *>(gam[1] + 32 * half + c0 + j);
      const float d[4] = {c.x, c.y, c.z, c.w}, dl[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float f = rowf * decay(gh, gl, d[e], dl[e]);
        x[j + e] = c0 + j + e <= last ? f * x[j + e] : 0.f;
      }
    }
    if (row < 64) {
#pragma unroll
      for (int j = 0; j < 16; j += 4)
        *reinterpret_cast<float4 *>(As + r64 * kLd + 32 * half + c0 + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
    } else {
      tmem_st16(taddr + c0, x);  // P waits there for the inverse
      if constexpr (!BF)
#pragma unroll
        for (int j = 0; j < 16; ++j) mp = max(mp, abs_bits(x[j]));
    }
  }
  if constexpr (!BF) {
    mp = __reduce_max_sync(0xffffffffu, mp);
    if ((tid & 31) == 0) atomicMax(&size[1], mp);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (tid < 64) {
    // column j of the inverse of diagonal block blk
    const int blk = tid >> 4, j = tid & 15, o = 16 * blk;
    float y[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s = i == j ? 1.f : 0.f;
#pragma unroll
      for (int m = 0; m < i; m += 4) {
        const float4 r = *reinterpret_cast<const float4 *>(As + (o + i) * kLd + o + m);
        s = fmaf(-r.x, y[m], s);
        if (m + 1 < i) s = fmaf(-r.y, y[m + 1], s);
        if (m + 2 < i) s = fmaf(-r.z, y[m + 2], s);
        if (m + 3 < i) s = fmaf(-r.w, y[m + 3], s);
      }
      y[i] = i < j ? 0.f : s;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) Ti[(o + i) * kLd + o + j] = y[i];
  } else {
    // the six 16 x 16 blocks above the diagonal blocks
    for (int e = tid - 64; e < 6 * 64; e += kPrepThreads - 64) {
      const int q = e >> 6, f = e & 63;
      const int bi = q < 3 ? 0 : (q < 5 ? 1 : 2), bj = q < 3 ? q + 1 : (q < 5 ? q - 1 : 3);
      *reinterpret_cast<float4 *>(Ti + (16 * bi + (f >> 2)) * kLd + 16 * bj + (f & 3) * 4) = make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }
  __syncthreads();
  inverse_level<16>(As, Ti);
  inverse_level<32>(As, Ti);
  float sP = 1.f;
  if constexpr (!BF) {
    float inv;
    sP = unit_of(size[1], &inv);
    if (tid == 0)
      *reinterpret_cast<float4 *>(a.w.unit + ch * kUnits) =
          make_float4(inv, fmaxf(1.f, __uint_as_float(size[0])), fmaxf(fabsf(a.p.scale), __uint_as_float(size[1])),
                      sqrtf(__uint_as_float(size[2])));
  }
  {
    // T and P as two-term tiles over the matrices: read, then (every thread being past its reads) written
    uint4 h[4], l[4];
#pragma unroll
    for (int c0 = 0; c0 < 2; ++c0) {
      float x[16];
      if (row < 64) {
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          const float4 r = *reinterpret_cast<const float4 *>(Ti + r64 * kLd + 32 * half + 16 * c0 + j);
          x[j] = r.x;
          x[j + 1] = r.y;
          x[j + 2] = r.z;
          x[j + 3] = r.w;
        }
      } else {
        tmem_ld16(taddr + 16 * c0, x);
        if constexpr (!BF)
#pragma unroll
          for (int j = 0; j < 16; ++j) x[j] *= sP;
      }
      split8<BF>(x, h[2 * c0], l[2 * c0]);
      split8<BF>(x + 8, h[2 * c0 + 1], l[2 * c0 + 1]);
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint32_t at = chunk_at(row, 4 * half + c);
      sts(sb + TT + at, h[c]);
      sts(sb + TT + 16384 + at, l[c]);
    }
  }
  publish();
  if (warp_leader()) {
    tc_fence_after();
    // rows 64..127: P T (rows 0..63, T T, are not read)
    const uint32_t id = idesc_f16(128, 64, BF, false, true);
    const KMajor ph_{sb + TT, 0}, pl{sb + TT + 16384, 0};
    const MNMajor th{sb + TT, 0}, tl{sb + TT + 16384, 0};
    issue<4>(tmem, ph_, th, id, false);
    issue<4>(tmem, ph_, tl, id, true);
    issue<4>(tmem, pl, th, id, true);
    mma_commit(smem_u32(&ctl.mma_bar));
  }
  wait_bar(ctl.mma_bar, ph, ctl, a.p.status);
  if (row >= 64) {
#pragma unroll
    for (int c0 = 0; c0 < 2; ++c0) {
      float x[16];
      tmem_ld16(taddr + 16 * c0, x);
      store_split16<BF>(sb + TT, sb + TT + 16384, row, 4 * half + 2 * c0, x);
    }
  }
  fence_async_smem();
  cta_end(tmem, 64);
  if (tid == 0) {
    bulk_store(a.w.T + ch * kImgT, sb + TT, kImgT);
    tma_store_commit();
    tma_store_wait_read0();
  }
}

// ------------------------------------------------------------- shared of the scans --
// Zeros for the rows of a packed batch that belong to no sequence: 64 columns of one head.
__device__ void zero_outside(const Args &a, const kda_tensor &o, int h, int col0) {
  const int lo = a.w.bound[0], hi = a.w.bound[a.nseq];
  const int64_t rows = (int64_t)lo + (a.p.T - hi);
  uint16_t *base = static_cast<uint16_t *>(o.data) + h * o.stride_h + col0;
  for (int64_t e = threadIdx.x; e < rows * 8; e += blockDim.x) {
    const int64_t r = e >> 3, t = r < lo ? r : r - lo + hi;
    *reinterpret_cast<uint4 *>(base + t * o.stride_t + (e & 7) * 8) = make_uint4(0, 0, 0, 0);
  }
}
__device__ void zero_outside(const Args &a, void *p, int dtype, int h) {
  const int lo = a.w.bound[0], hi = a.w.bound[a.nseq];
  const int64_t rows = (int64_t)lo + (a.p.T - hi);
  for (int64_t r = threadIdx.x; r < rows; r += blockDim.x)
    store_gate(p, (int64_t)h * a.p.T + (r < lo ? r : r - lo + hi), dtype, 0.f);
}

// ------------------------------------------------------------------ the scans --
// The state is transposed in tensor memory:
// lanes are the value channels, columns the key channels, so that the operand that changes
// from step to step (the state, X, U) is always the first one and goes from registers
// straight back into tensor memory, split in two terms, without touching shared memory:
//   forward   [K S]^T = S^T K^T      X^T          U^T = X^T T^T          S^T += U'^T K
//   reverse   [K dS]^T = dS^T K^T    Z^T          dX^T = Z^T T + dO^T PT dS^T += dY^T K + dO^T Q'
// (U' = e^{gamma_63 - gamma} U, dY = -G beta dX, Q' = scale G Q).  A first version with the
// state as the second operand in shared memory spent 880 of 6750 cycles a chunk and half
// state on the first product alone: its operands, not its arithmetic, set the time.
//
// Scheduling.  The chunks of all streams (sequence, head), stream after stream, are cut into as
// many equal ranges as there are CTAs (one an SM), so that 160 streams on 148 SMs take 35 chunks'
// time and not 64.  The state crosses a cut through a slot in global memory.  A CTA first runs the
// piece that ends its range, which begins a stream and waits for nobody, and publishes its state;
// the piece that begins its range, whose first state is the one that the range before published
// first of all, comes last.  Ranges go by tickets, so a CTA only waits for one that is running.
//
// Warps: 8 walk the dependent chain (a value channel a thread, half the columns each), 4
// turn finished tiles into output or workspace rows, one starts the loads, one issues the
// products.  TMA brings the tiles two chunks ahead.  In fp16 two more warps find each chunk's unit.
//
// Measured at D = 128: 2.5 us a chunk (4600 cycles) with outputs, whatever the number of streams up
// to one an SM (28 streams of 32768 tokens: 1.29 ms).  It is latency: three dependent products with a
// tensor-memory round trip, a conversion to two terms and two barriers each (state conversion 970 cycles, K S 820,
// X 540, T X 610, U 620, update 650).  16 x 2048 tokens of 10 heads (160 streams on 148 SMs): outputs 118 us
// (503 MB, 4.3 TB/s), states and u rows 148 us (755 MB, 5.1 TB/s), reverse 199 us (983 MB, 4.9 TB/s; its start
// under the end of the one before is in that).  dO becomes an operand in the chain's wait for its
// product with T: in the output warps that took 2000 to 3000 cycles a chunk and made them the slowest.
// fp16's units cost a chunk 1000 cycles of the chain (its maximum as the state is converted, the wait for
// the unit): 28 streams of 32768 tokens 1.57 ms, and 171, 174 and 305 us in place of 118, 148 and 199.
// With the sizes found by the chain itself (the state read twice, a barrier) the former took 1.63 ms.
enum { kOut = 0, kStore = 1, kRev = 2 };  // outputs; state and u rows for the backward; reverse scan

template <bool BF>
constexpr int kScanThreads = BF ? 448 : 512;
constexpr int kOutWarp = 8, kLoadWarp = 12, kMmaWarp = 13, kSizeWarp = 14;  // the chain: warps 0 .. 7; fp16: two size warps

// Per-token factors of a chunk, one array a factor: beta, -beta e^gamma, e^{gamma_63 - gamma}, scale e^gamma.
struct Factors {
  float beta[64], bg[64], w[64], sg[64];
  float last[4];  // e^{gamma_63}; fp16's reverse scan: the power of two that is taken out of it and of bg and sg
  float4 unit;    // fp16: the preparation's four sizes
};

template <int D, int MODE>
struct ScanSmem {
  static constexpr uint32_t kTile = 64 * D * 2;  // [64 tokens x D], D / 64 swizzled blocks of 8 KB
  static constexpr uint32_t K = 0, Q = kTile, V = 2 * kTile, T = 3 * kTile, kStage = T + kImgT;
  static constexpr uint32_t OUT = 2 * kStage;  // outputs: o; reverse: dX hi, dX lo, dV
  static constexpr uint32_t kBytes = OUT + (MODE == kOut ? kTile : (MODE == kRev ? 3 * kTile : 0));
};

struct ScanBars {
  uint64_t full[2], empty[2];
  uint64_t tail[2], s_ready[2], inputs_sized[2], state_sized[2], unit_ready[2], ks_done, x_ready, u_done, up_ready, s_done, o_done, out_free, qs_ready;
};

// Wait (bounded, like mbar_wait) for a range's entry state.
__device__ __forceinline__ void wait_flag(const int *flag, int32_t *status, volatile int *abort_flag) {
  if ((threadIdx.x & 31) == 0) {
    const long long t0 = clock64();
    int v = 0;
    while (!*abort_flag) {
      asm volatile("ld.acquire.gpu.global.b32 %0, [%1];" : "=r"(v) : "l"(flag) : "memory");
      if (v != 0) break;
      if (clock64() - t0 > kWaitCycles) {
        if (status) atomicOr(status, KDA_ERR_DEVICE_TIMEOUT);
        *abort_flag = 1;
      }
    }
    __threadfence();
  }
  __syncwarp();
}

__device__ __forceinline__ Streams streams_of(const Args &a) {
  return {a.p.cu_seqlens == nullptr ? nullptr : a.w.first, a.per_seq, a.nseq, a.p.H};
}
// Each warp keeps its place in shared memory: as registers of every thread it made the chain spill.
struct WarpPlace {
  Pieces pieces;
  Piece pc;
  Seq s;
  int more;
};

// tensor-memory columns
constexpr uint32_t cS = 0, cSH = 128, cSL = 192, cXH = 256, cXL = 288, cR1 = 320, cR2 = 384, cR3 = 448;

// 32 fp32 columns as two 16-column tiles of packed pairs in tensor memory
template <bool BF>
__device__ __forceinline__ void tmem_split32(uint32_t hi_at, uint32_t lo_at, const float (&x)[32]) {
  uint32_t h[16], l[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) split2<BF>(x[2 * i], x[2 * i + 1], h[i], l[i]);
  tmem_st_32x32b_x16_nowait(hi_at, h);
  tmem_st_32x32b_x16_nowait(lo_at, l);
}

__device__ __forceinline__ void stmatrix_x4_trans(uint32_t addr, uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(r0), "r"(r1), "r"(r2),
               "r"(r3)
               : "memory");
}

// 16 x 256b fragments (64 columns of 16 lanes) times a per-column factor, rounded and stored
// transposed: rows of the swizzled tile are columns (tokens), 16-byte runs are lanes (value channels).
struct TileOut {
  int quad, mat, rho;
  __device__ __forceinline__ explicit TileOut(int quad_) : quad(quad_), mat((threadIdx.x & 31) >> 3), rho(threadIdx.x & 7) {}
  __device__ __forceinline__ void put(uint32_t tile, int hh, int j, uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3) const {
    const int m0 = 32 * quad + 16 * hh + 8 * (mat & 1), tok = 8 * (j + (mat >> 1)) + rho;
    stmatrix_x4_trans(tile + (uint32_t)((m0 >> 6) * 8192) + chunk_at(tok, (m0 & 63) >> 3), r0, r1, r2, r3);
  }
};

// TMA maps of a scan: k, q, v (reverse: dout), o (reverse: dv)
struct Maps {
  CUtensorMap k, q, v, o;
};

// `block`: this CTA's number among the scan's
template <int D, bool BF, int MODE>
__device__ __forceinline__ void scan_cta(const Args &a, const Maps &maps, int block) {
  using L = ScanSmem<D, MODE>;
  constexpr int Q = D / 32;  // warps that own live tensor-memory lanes, of four
  constexpr int NB = D / 64;
  constexpr bool REV = MODE == kRev;
  extern __shared__ __align__(1024) char smem[];
  __shared__ ScanBars bars;
  __shared__ __align__(16) Factors fac[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  __shared__ WarpPlace places[kScanThreads<BF> / 32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G_ = a.p.H / a.p.Hk;
  pdl_wait();
  if (MODE != kStore) {
    if (a.p.cu_seqlens != nullptr)  // the rows outside all sequences
      for (int h = block; h < a.p.H; h += a.ranges) {
        for (int c = 0; c < D; c += 64) {
          if (MODE == kOut) zero_outside(a, a.p.o, h, c);
          if (REV) {
            zero_outside(a, a.p.dv, h, c);
            if (h % G_ == 0) {
              zero_outside(a, a.p.dq, h / G_, c);
              zero_outside(a, a.p.dk, h / G_, c);
            }
          }
        }
        if (REV) {
          zero_outside(a, a.p.dg, a.p.g_dtype, h);
          zero_outside(a, a.p.dbeta, a.p.beta_dtype, h);
        }
      }
    const float *src = REV ? a.p.dstate_out : a.p.state_in;
    float *dst = REV ? a.p.dstate_in : a.p.state_out;
    if (dst != nullptr)  // sequences without tokens hand their state on
      for (int i = block; i < a.nseq * a.p.H; i += a.ranges)
        if (get_seq(a, i / a.p.H).len == 0)
          for (int e = tid; e < D * D; e += kScanThreads<BF>) dst[(size_t)i * D * D + e] = src != nullptr ? src[(size_t)i * D * D + e] : 0.f;
  }
  __shared__ int range_slot;
  // fp16, by chunk parity: a warp of the chain each, the largest element that is left of the state before the chunk
  // and of what half the tokens added to it; the second sizing warp's part of the inputs' sizes
  __shared__ float2 sizes[2][8];
  __shared__ uint2 part_size[2];
  __shared__ float units[2][3];     // fp16: a chunk's unit, its inverse, what its dO adds to dS at most
  int *queue = a.w.queue + (REV ? a.ranges + 2 : 0);
  float *slots = a.w.slots + (REV ? (size_t)(a.ranges + 1) * D * D : 0);
  float2 *cuts = BF ? nullptr : a.w.cuts + (REV ? 8 * (a.ranges + 1) : 0);
  const uint32_t sb = smem_u32(smem);
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&bars.full[i]), 32);
      mbar_init(smem_u32(&bars.empty[i]), MODE == kStore ? 1 : 1 + Q);
      mbar_init(smem_u32(&bars.s_ready[i]), 2 * Q);
      mbar_init(smem_u32(&bars.tail[i]), 32);
      mbar_init(smem_u32(&bars.inputs_sized[i]), 1);
      mbar_init(smem_u32(&bars.state_sized[i]), 2 * Q);
      mbar_init(smem_u32(&bars.unit_ready[i]), 1);
    }
    for (uint64_t *b : {&bars.x_ready, &bars.up_ready}) mbar_init(smem_u32(b), 2 * Q);
    for (uint64_t *b : {&bars.ks_done, &bars.u_done, &bars.s_done, &bars.o_done}) mbar_init(smem_u32(b), 1);
    mbar_init(smem_u32(&bars.out_free), Q);
    mbar_init(smem_u32(&bars.qs_ready), 2 * Q);
    mbar_fence_init();
    abort_flag = 0;
    // ranges that are whole streams need no order
    range_slot = a.p.cu_seqlens == nullptr && a.ranges == a.nseq * a.p.H ? block : (a.max_chunks > 0 ? atomicAdd(queue, 1) : 0);
  }
  if (warp == kMmaWarp) {
    tmem_alloc(smem_u32(&tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(&tmem_slot);
  auto wait = [&](uint64_t &b, uint32_t parity) {
    mbar_wait(smem_u32(&b), parity, a.p.status, &abort_flag);
    __syncwarp();
  };
  auto arrive_warp = [&](uint64_t &b) {  // after this warp's tensor-memory accesses
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&b));
  };

  pdl_launch_dependents();
  const int range = *reinterpret_cast<volatile int *>(&range_slot);
  int lo, hi;
  range_of(a.max_chunks == 0 ? 0 : streams_of(a).total(), a.ranges, range, &lo, &hi);
  WarpPlace &place = places[warp];
  if (lane == 0) place.pieces.begin(streams_of(a), lo, hi);
  const Piece &pc = place.pc;
  const Seq &s = place.s;
  auto step_piece = [&]() {  // one lane
    place.more = place.pieces.next(streams_of(a), &place.pc);
    if (place.more) place.s = get_seq(a, place.pc.n);
  };
  int p0 = 0, p1 = 0, rp = -1;  // the piece's positions, and that of its stream's ragged chunk
  auto take_piece = [&]() {
    if (*reinterpret_cast<volatile int *>(&place.more) == 0) return false;
    p0 = pc.p0;
    p1 = pc.p1;
    rp = s.len % kChunk == 0 ? -1 : (REV ? 0 : pc.nc - 1);
    return true;
  };
  auto next_piece = [&]() {
    __syncwarp();
    if (lane == 0) step_piece();
    __syncwarp();
    return take_piece();
  };
  // of position `pos` of the current piece's stream
  auto chunk_of = [&](int pos) { return REV ? pc.nc - 1 - pos : pos; };
  auto cell = [&](int pos) { return (size_t)(s.chunk0 + chunk_of(pos)) * a.p.H + pc.h; };
  auto rows_of = [&](int pos) { return min(kChunk, s.len - chunk_of(pos) * kChunk); };
  // Every role counts the chunks that it has begun, over all pieces (it: stages and barrier phases), and
  // keeps the phases of the stages' tail barriers, which ragged chunks alone complete (bits of tails).
  int it = 0, tails = 0;
  auto wait_tail = [&](int st) {
    mbar_wait(smem_u32(&bars.tail[st]), (tails >> st) & 1, a.p.status, &abort_flag);
    tails ^= 1 << st;
  };
  // a stage's tiles have landed (and, in a sequence's ragged chunk, the rows behind its end are zeros)
  auto wait_full = [&](int pos) {
    wait(bars.full[it & 1], (it >> 1) & 1);
    if (pos == rp) {
      wait_tail(it & 1);
      __syncwarp();
    }
  };

  if (warp < kOutWarp) {
    // ------------------------------------------------------------- the chain --
    const int quad = warp & 3, half = warp >> 2;
    if (quad < Q) {
      const uint32_t tl = tmem + ((uint32_t)quad << 21);
      const int dv = 32 * quad + lane;
      constexpr int W = D / 2;  // key channels of this thread
      const size_t own = (size_t)(half * W) * D + dv;  // this thread's first element of a [D][D] state
      // byte offsets of column dv in rows t = 0..7 of a swizzled tile
      uint32_t vcol[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) vcol[i] = (uint32_t)((dv >> 6) * 8192 + i * 128 + ((((dv >> 3) ^ i) & 7) << 4) + (dv & 7) * 2);
      // what chunk i's unit goes by: what is left of the state before the last chunk, what half of its tokens added
      auto tell_size = [&](int i, float2 z) {
        if (lane == 0) {
          sizes[i & 1][half * Q + quad] = z;
          mbar_arrive(smem_u32(&bars.state_sized[i & 1]));
        }
      };
      while (next_piece()) {
        const size_t state = ((size_t)pc.n * a.p.H + pc.h) * D * D;
        // the piece's first state: the caller's, or the one that the range before published
        const float *src = REV ? a.p.dstate_out : a.p.state_in;
        if (src != nullptr) src += state;
        if (pc.p0 > 0) {
          wait_flag(queue + 1 + range, a.p.status, &abort_flag);
          src = slots + (size_t)range * D * D;
        }
        float unit = 1.f, worth = 1.f;  // fp16: of the state in tensor memory (a first state comes as it is)
        for (int pos = p0; pos < p1; ++pos, ++it) {
          const int st = it & 1;
          wait_full(pos);
          const float last = fac[st].last[0];
          if (!BF && pos == p0) {  // fp16: how large a piece's first state is
            if (pc.p0 > 0) {  // what the chunk before said of it: units do not depend on where streams are cut
              tell_size(it, __ldcg(cuts + 8 * range + half * Q + quad));
            } else {
              uint32_t m = 0;
              if (src != nullptr)
#pragma unroll 8
                for (int j = 0; j < W; ++j) m = max(m, abs_bits(__ldcg(src + own + (size_t)j * D)));
              tell_size(it, make_float2(__uint_as_float(__reduce_max_sync(0xffffffffu, m)), 0.f));
            }
          }
          if (it > 0) {
            if (MODE != kOut) wait(bars.out_free, (it - 1) & 1);
            wait(bars.s_done, (it - 1) & 1);
          }
          tc_fence_after();
          float held = 1.f, large = 0.f;  // fp16: new units of an old one; of the state that the chunk begins with, in its units
          if constexpr (!BF) {
            wait(bars.unit_ready[st], (it >> 1) & 1);
            unit = units[st][0];
            held = fminf(worth * unit, 0x1p126f);  // beyond that nothing is left of what is held
            worth = REV ? units[st][1] * fac[st].last[1] : units[st][1];
          }
#pragma unroll
          for (int c0 = 0; c0 < W; c0 += 32) {
            float x[32];
            if (pos > p0) {
              tmem_ld32(tl + cS + half * W + c0, x);
            } else {
#pragma unroll
              for (int j = 0; j < 32; ++j) x[j] = src != nullptr ? __ldcg(src + own + (size_t)(c0 + j) * D) : 0.f;
            }
            if constexpr (!BF) {
              if (held != 1.f)
#pragma unroll
                for (int j = 0; j < 32; ++j) x[j] *= held;
              float m[4] = {large, 0.f, 0.f, 0.f};
#pragma unroll
              for (int j = 0; j < 32; ++j) m[j & 3] = fmaxf(m[j & 3], fabsf(x[j]));
              large = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
            }
            tmem_split32<BF>(tl + cSH + (half * W + c0) / 2, tl + cSL + (half * W + c0) / 2, x);
            uint32_t r[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(x[j] * last);
            tmem_st_32x32b_x32_nowait(tl + cS + half * W + c0, r);
            tmem_wait_st();
            arrive_warp(bars.s_ready[c0 / 32]);
          }
          float v[32];
          if (!REV) {  // V^T: this value channel of 32 tokens
            const uint32_t vt = sb + st * L::kStage + L::V + half * 4096;
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              uint16_t u;
              asm volatile("ld.shared.u16 %0, [%1];" : "=h"(u) : "r"(vt + vcol[j & 7] + (j >> 3) * 1024));
              v[j] = unpack2((uint32_t)u, BF).x * fac[st].beta[32 * half + j];
              if constexpr (!BF) v[j] *= unit;
            }
          }
          wait(bars.ks_done, it & 1);
          tc_fence_after();
          {
            float x[32];
            tmem_ld32(tl + cR1 + 32 * half, x);
#pragma unroll
            for (int j = 0; j < 32; ++j) x[j] = REV ? fac[st].w[32 * half + j] * x[j] : fmaf(fac[st].bg[32 * half + j], x[j], v[j]);
            tmem_split32<BF>(tl + cXH + 16 * half, tl + cXL + 16 * half, x);
            tmem_wait_st();
            arrive_warp(bars.x_ready);
          }
          if (REV) {  // Q' product's first operand, scale e^gamma dO transposed, under the product with T
            const uint32_t vt = sb + st * L::kStage + L::V + half * 4096;
            float x[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              uint16_t u;
              asm volatile("ld.shared.u16 %0, [%1];" : "=h"(u) : "r"(vt + vcol[j & 7] + (j >> 3) * 1024));
              x[j] = unpack2((uint32_t)u, BF).x * fac[st].sg[32 * half + j];
              if constexpr (!BF) x[j] *= unit;
            }
            tmem_split32<BF>(tl + cR3 + 16 * half, tl + cR3 + 32 + 16 * half, x);
            tmem_wait_st();
            arrive_warp(bars.qs_ready);
          }
          wait(bars.u_done, it & 1);
          tc_fence_after();
          {
            float x[32];
            tmem_ld32(tl + (REV && BF ? cR2 : cR1) + 32 * half, x);
            if constexpr (REV && !BF) {  // fp16: dO's part is in P T's unit
              float y[32];
              tmem_ld32(tl + cR2 + 32 * half, y);
              const float f = fac[st].unit.x * unit;
#pragma unroll
              for (int j = 0; j < 32; ++j) x[j] = fmaf(f, y[j], x[j]);
            }
#pragma unroll
            for (int j = 0; j < 32; ++j) x[j] *= REV ? fac[st].bg[32 * half + j] : fac[st].w[32 * half + j];
            // over an operand whose products are done: S^T's (outputs: X^T may still be in use), else X^T's
            const uint32_t at = MODE == kOut ? cSH : cXH;
            tmem_split32<BF>(tl + at + 16 * half, tl + at + 32 + 16 * half, x);
            tmem_wait_st();
            const float kn = BF ? 0.f : fac[st].unit.w;
            arrive_warp(bars.up_ready);
            if constexpr (!BF) {  // under the update: |sum_t k_t u'_t| <= max |k_t| sum_t |u'_t|
              float g4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int j = 0; j < 32; ++j) g4[j & 3] += fabsf(x[j]);
              const float g = (g4[0] + g4[1]) + (g4[2] + g4[3]);
              const float2 z = make_float2(__uint_as_float(__reduce_max_sync(0xffffffffu, abs_bits(large))) * last * worth + (REV ? units[st][2] : 0.f),
                                           __uint_as_float(__reduce_max_sync(0xffffffffu, abs_bits(g))) * kn * worth);
              if (pos + 1 < p1)
                tell_size(it + 1, z);
              else if (pc.p1 < pc.nc && lane == 0)
                __stcg(cuts + 8 * (range + 1) + half * Q + quad, z);
            }
          }
        }
        // where the state goes from here: to the next range, or to the caller
        float *dst = pc.p1 < pc.nc ? slots + (size_t)(range + 1) * D * D
                                   : (REV ? a.p.dstate_in : (MODE == kOut ? a.p.state_out : nullptr));
        if (dst != nullptr) {
          if (pc.p1 == pc.nc) dst += state;
          wait(bars.s_done, (it - 1) & 1);
          tc_fence_after();
#pragma unroll
          for (int c0 = 0; c0 < W; c0 += 32) {
            float x[32];
            tmem_ld32(tl + cS + half * W + c0, x);
#pragma unroll
            for (int j = 0; j < 32; ++j) __stcg(dst + own + (size_t)(c0 + j) * D, BF ? x[j] : x[j] * worth);
          }
          if (pc.p1 < pc.nc) {
            __threadfence();
            named_bar_sync(2, 2 * Q * 32);
            if (warp == 0 && lane == 0) {
              __threadfence();
              atomicExch(queue + 2 + range, 1);
            }
          }
        }
      }
    }
  } else if (warp < kLoadWarp) {
    // ------------------------------------------------------ finished tiles out --
    const int quad = warp & 3;
    if (quad < Q) {
      const uint32_t tl = tmem + ((uint32_t)quad << 21);
      const int t = tid - kOutWarp * 32;  // 0 .. 32 Q - 1
      const int row = 32 * quad + lane, q2 = 2 * (lane & 3);
      const TileOut tile(quad);
      const kda_tensor &ot = REV ? a.p.dv : a.p.o;
      // a [64 x D] tile of o or dV from shared memory, once all warps have written it (store_tile ends the wait
      // for its reads; the caller's next tile starts with tile_free)
      auto store_tile = [&](uint32_t at, int pos) {
        const int c = chunk_of(pos), rows = rows_of(pos);
        fence_async_smem();
        named_bar_sync(1, 32 * Q);
        if (rows == kChunk) {
          if (t == 0)
            for (int b = 0; b < NB; ++b) tma_store_4d(&maps.o, at + 8192 * b, 64 * b, (int)(s.t0 + (int64_t)c * kChunk), pc.h, (int)s.b);
        } else {  // what lies behind a packed sequence is another's
          uint16_t *ob = static_cast<uint16_t *>(ot.data) + s.b * ot.stride_b + pc.h * ot.stride_h + (s.t0 + (int64_t)c * kChunk) * ot.stride_t;
          for (int e = t; e < rows * (D / 8); e += 32 * Q) {
            const int r = e / (D / 8), g = e % (D / 8);
            *reinterpret_cast<uint4 *>(ob + r * ot.stride_t + 8 * g) = ld_shared_v4(at + (g >> 3) * 8192 + chunk_at(r, g & 7));
          }
        }
      };
      auto tile_free = [&]() {
        if (t == 0) tma_store_wait_read0();
        named_bar_sync(1, 32 * Q);
      };
      // fp16: the chunk's unit and its inverse
      auto unit_at = [&](float *worth) {
        if (BF) return *worth = 1.f;
        wait(bars.unit_ready[it & 1], (it >> 1) & 1);
        *worth = units[it & 1][1];
        return units[it & 1][0];
      };
      while (next_piece()) {
        for (int pos = p0; pos < p1; ++pos, ++it) {
          const int st = it & 1;
          float worth;
          const float unit = unit_at(&worth);
          if (MODE == kOut) {
            wait_full(pos);
            wait(bars.o_done, it & 1);
            tc_fence_after();
            const float of = BF ? 1.f : fac[st].unit.x * worth;
            uint32_t pk[2][16];  // [16-lane half][column block j, row half]
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
              uint32_t qs[32], o[32];
              tmem_ld_16x256b_x8(tl + ((uint32_t)(16 * hh) << 16) + cR2, qs);
              tmem_ld_16x256b_x8(tl + ((uint32_t)(16 * hh) << 16) + cR3, o);
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                float f0 = fac[st].sg[8 * j + q2], f1 = fac[st].sg[8 * j + q2 + 1];
                if constexpr (!BF) {
                  f0 *= worth;
                  f1 *= worth;
#pragma unroll
                  for (int e = 0; e < 4; ++e) o[4 * j + e] = __float_as_uint(__uint_as_float(o[4 * j + e]) * of);
                }
#pragma unroll
                for (int e = 0; e < 2; ++e)
                  pk[hh][2 * j + e] = pack2(fmaf(f0, __uint_as_float(qs[4 * j + 2 * e]), __uint_as_float(o[4 * j + 2 * e])),
                                            fmaf(f1, __uint_as_float(qs[4 * j + 2 * e + 1]), __uint_as_float(o[4 * j + 2 * e + 1])), BF);
              }
            }
            arrive_warp(bars.out_free);
            if (lane == 0) mbar_arrive(smem_u32(&bars.empty[st]));
            tile_free();
#pragma unroll
            for (int hh = 0; hh < 2; ++hh)
#pragma unroll
              for (int j = 0; j < 8; j += 2)
                tile.put(sb + L::OUT, hh, j, pk[hh][2 * j], pk[hh][2 * j + 1], pk[hh][2 * j + 2], pk[hh][2 * j + 3]);
            store_tile(sb + L::OUT, pos);
            if (t == 0) tma_store_commit();
          } else {
            if (REV) wait_full(pos);  // for the factors
            if (!BF && t == 0) a.w.unit[cell(pos) * kUnits + (REV ? kUnitR : kUnitF)] = worth;
          // the state (reverse: its gradient) as the chain split it
            char *img = (REV ? a.w.dS : a.w.S) + cell(pos) * (size_t)(D * D * 4) + row * 16;
#pragma unroll
            for (int b = 0; b < NB; ++b) wait(bars.s_ready[b], it & 1);
            tc_fence_after();
#pragma unroll
            for (int part = 0; part < 2; ++part)
#pragma unroll
              for (int b = 0; b < NB; ++b) {
                uint32_t r[32];
                tmem_ld_32x32b_x32(tl + (part ? cSL : cSH) + 32 * b, r);
#pragma unroll
                for (int g = 0; g < 8; ++g)
                  *reinterpret_cast<uint4 *>(img + part * (D * D * 2) + (8 * b + g) * (D * 16)) =
                      make_uint4(r[4 * g], r[4 * g + 1], r[4 * g + 2], r[4 * g + 3]);
              }
            wait(bars.u_done, it & 1);
            tc_fence_after();
            if (MODE == kStore) {  // U^T
              char *ui = a.w.U + cell(pos) * (size_t)(D * 256) + row * 16;
#pragma unroll
              for (int b = 0; b < 2; ++b) {
                float x[32];
                tmem_ld32(tl + cR1 + 32 * b, x);
                if (b == 1) arrive_warp(bars.out_free);
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                  uint4 hi, lo;
                  split8<BF>(x + 8 * g, hi, lo);
                  *reinterpret_cast<uint4 *>(ui + (4 * b + g) * (D * 16)) = hi;
                  *reinterpret_cast<uint4 *>(ui + D * 128 + (4 * b + g) * (D * 16)) = lo;
                }
              }
            } else {  // dX, and dV = beta dX
              tile_free();
#pragma unroll
              for (int hh = 0; hh < 2; ++hh) {
                uint32_t x[32], hi[16], lo[16];
                tmem_ld_16x256b_x8(tl + ((uint32_t)(16 * hh) << 16) + cR2, x);
                if constexpr (!BF) {
                  uint32_t z[32];
                  tmem_ld_16x256b_x8(tl + ((uint32_t)(16 * hh) << 16) + cR1, z);
                  const float f = fac[st].unit.x * unit;
#pragma unroll
                  for (int i = 0; i < 32; ++i) x[i] = __float_as_uint(fmaf(f, __uint_as_float(x[i]), __uint_as_float(z[i])));
                }
                if (hh == 1) arrive_warp(bars.out_free);
#pragma unroll
                for (int i = 0; i < 16; ++i) split2<BF>(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1]), hi[i], lo[i]);
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                  tile.put(sb + L::OUT, hh, j, hi[2 * j], hi[2 * j + 1], hi[2 * j + 2], hi[2 * j + 3]);
                  tile.put(sb + L::OUT + L::kTile, hh, j, lo[2 * j], lo[2 * j + 1], lo[2 * j + 2], lo[2 * j + 3]);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                  float f0 = fac[st].beta[8 * j + q2], f1 = fac[st].beta[8 * j + q2 + 1];
                  if constexpr (!BF) {
                    f0 *= worth;
                    f1 *= worth;
                  }
#pragma unroll
                  for (int e = 0; e < 2; ++e)
                    hi[2 * j + e] = pack2(f0 * __uint_as_float(x[4 * j + 2 * e]), f1 * __uint_as_float(x[4 * j + 2 * e + 1]), BF);
                }
#pragma unroll
                for (int j = 0; j < 8; j += 2)
                  tile.put(sb + L::OUT + 2 * L::kTile, hh, j, hi[2 * j], hi[2 * j + 1], hi[2 * j + 2], hi[2 * j + 3]);
              }
              __syncwarp();
              if (lane == 0) mbar_arrive(smem_u32(&bars.empty[st]));
              store_tile(sb + L::OUT + 2 * L::kTile, pos);
              if (t == 0) {  // the dX tiles are the images
                char *xi = a.w.dX + cell(pos) * (size_t)(D * 256);
                for (int b = 0; b < NB; ++b) {
                  bulk_store(xi + b * 16384, sb + L::OUT + b * 8192, 8192);
                  bulk_store(xi + b * 16384 + 8192, sb + L::OUT + L::kTile + b * 8192, 8192);
                }
                tma_store_commit();
              }
            }
          }
        }
      }
      if (t == 0) tma_store_wait_all();
    }
  } else if (warp == kLoadWarp) {
    // ------------------------------------------------------------------ loads --
    constexpr uint32_t kBytes = (MODE == kStore ? 2 : 3) * L::kTile + (MODE == kStore ? 16384 : kImgT);
    auto load = [&](int pos) {
      const int st = it & 1;
      const uint32_t base = sb + st * L::kStage, bar = smem_u32(&bars.full[st]);
      const size_t at = cell(pos) * 64;
      const float *gam = a.w.gam + 2 * at;
      float4 unit;
      float lh, ll, gh[2], gl[2], be[2];
      auto fetch = [&]() {
        lh = gam[63];
        ll = gam[127];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          gh[i] = gam[lane + 32 * i];
          gl[i] = gam[64 + lane + 32 * i];
          be[i] = a.w.beta[at + lane + 32 * i];
        }
      };
      if constexpr (!BF) {  // (the sizes of the chunk need the time behind the tiles)
        unit = *reinterpret_cast<const float4 *>(a.w.unit + cell(pos) * kUnits);
        fetch();
      }
      if (it >= 2) wait(bars.empty[st], ((it >> 1) - 1) & 1);
      if (lane == 0) {
        const int t0 = (int)(s.t0 + (int64_t)chunk_of(pos) * kChunk), b = (int)s.b;
        mbar_expect_tx(bar, kBytes);
        for (int i = 0; i < NB; ++i) {
          tma_load_4d(base + L::K + 8192 * i, &maps.k, bar, 64 * i, t0, pc.h / G_, b);
          if (MODE != kStore) tma_load_4d(base + L::Q + 8192 * i, &maps.q, bar, 64 * i, t0, pc.h / G_, b);
          tma_load_4d(base + L::V + 8192 * i, &maps.v, bar, 64 * i, t0, pc.h, b);
        }
        const char *img = a.w.T + cell(pos) * kImgT;
        if (MODE == kStore) {  // T alone
          bulk_load(base + L::T, img, 8192, bar);
          bulk_load(base + L::T + 16384, img + 16384, 8192, bar);
        } else {
          bulk_load(base + L::T, img, kImgT, bar);
        }
      }
      if constexpr (BF) fetch();
      // All that the reverse scan hands on has a factor e^gamma of its token, at most the first one's (g <= 0): fp16
      // takes its power of two out before it splits, and back in with the unit.
      float out = 1.f, rest = 1.f;
      if constexpr (REV && !BF) {
        const float most = ex2f(fminf(__shfl_sync(0xffffffffu, gh[0], 0), 0.f));
        rest = __uint_as_float(max(__float_as_uint(most) >> 23, 67u) << 23);  // 2^-60 at least
        out = __uint_as_float((254u << 23) - __float_as_uint(rest));
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float G = ex2f(gh[i]);
        if constexpr (REV && !BF) G *= out;
        fac[st].beta[lane + 32 * i] = be[i];
        fac[st].bg[lane + 32 * i] = -be[i] * G;
        fac[st].w[lane + 32 * i] = decay(lh, ll, gh[i], gl[i]);
        fac[st].sg[lane + 32 * i] = a.p.scale * G;
      }
      if (lane == 0) {
        fac[st].last[0] = REV && !BF ? ex2f(lh) * out : ex2f(lh);
        if constexpr (REV && !BF) fac[st].last[1] = rest;
        if constexpr (!BF) fac[st].unit = unit;
      }
      mbar_arrive(bar);
      __syncwarp();
    };
    // a ragged chunk once it has landed: zeros behind its end
    auto zero_tail = [&](int st, int phase, int rows) {
      wait(bars.full[st], phase);
      for (int tl = 0; tl < 3; ++tl) {
        if (MODE == kStore && tl == 1) continue;
        const uint32_t base = sb + st * L::kStage + tl * L::kTile;
        for (int e = lane; e < (kChunk - rows) * (D / 8); e += 32) {
          const int r = rows + e / (D / 8), g = e % (D / 8);
          sts(base + (g >> 3) * 8192 + chunk_at(r, g & 7), make_uint4(0, 0, 0, 0));
        }
      }
      fence_async_smem();
      mbar_arrive(smem_u32(&bars.tail[st]));
    };
    int ragged = kChunk;  // rows of the chunk before
    while (next_piece()) {
      for (int pos = p0; pos < p1; ++pos, ++it) {
        load(pos);
        if (ragged < kChunk) zero_tail((it - 1) & 1, ((it - 1) >> 1) & 1, ragged);
        ragged = rows_of(pos);
      }
    }
    if (ragged < kChunk) zero_tail((it - 1) & 1, ((it - 1) >> 1) & 1, ragged);
  } else if (!BF && warp >= kSizeWarp) {
    // -------------------------------------------------------- fp16: the chunks' units --
    // From the inputs' largest elements and a bound of the state's: |S + sum_t k_t u'_t| <= |S| + max |k_t| sum_t |u'_t|
    // (exact for a piece's first state).  The chain gives its part before the update is done, and this is done before
    // it has to wait.  Two warps, eight rows of the tiles in turn, in a loop of few instructions: unrolled,
    // code that a warp runs once a chunk waits thousands of cycles to be fetched.
    constexpr int P = D / 8, RW = 32 / P, NL = 8 / RW;  // 16-byte pieces a row, rows a load, loads for eight rows
    const int second = warp - kSizeWarp;
    uint32_t off[NL];
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int r = lane / P + RW * i, g = lane % P;
      off[i] = (g >> 3) * 8192 + chunk_at(r, g & 7) + 1024 * second;
    }
    while (next_piece()) {
      for (int pos = p0; pos < p1; ++pos, ++it) {
        const int st = it & 1, rows = rows_of(pos);  // what lies behind a sequence's end is another's
        wait(bars.full[st], (it >> 1) & 1);
        uint32_t m[2] = {0, 0};
#pragma unroll
        for (int tl = 0; tl < (REV ? 2 : 1); ++tl) {
          const char *base = smem + st * L::kStage + (tl == 0 ? L::V : L::Q);
#pragma unroll 1
          for (int r0 = lane / P + 8 * second; r0 < rows; r0 += 16, base += 2048) {
            uint4 x[NL];
#pragma unroll
            for (int i = 0; i < NL; ++i) x[i] = *reinterpret_cast<const uint4 *>(base + off[i]);
#pragma unroll
            for (int i = 0; i < NL; ++i) m[tl] = max(m[tl], r0 + RW * i < rows ? half_size(x[i]) : 0u);
          }
          __syncwarp();
          m[tl] = __reduce_max_sync(0xffffffffu, m[tl]);
        }
        if (second) {
          if (lane == 0) {
            part_size[st] = make_uint2(m[0], m[1]);
            mbar_arrive(smem_u32(&bars.inputs_sized[st]));
          }
          __syncwarp();
          continue;
        }
        wait(bars.inputs_sized[st], (it >> 1) & 1);
        const uint2 other = part_size[st];
        const float x = unpack2(max(m[0], other.x), false).x, q = unpack2(max(m[1], other.y), false).x;
        const float inputs = x * fac[st].unit.y * (REV ? fac[st].unit.z : 1.f);
        wait(bars.state_sized[st], (it >> 1) & 1);
        const float2 z = sizes[st][lane & (2 * Q - 1)];
        const uint32_t left = __reduce_max_sync(0xffffffffu, abs_bits(z.x)), grown = __reduce_max_sync(0xffffffffu, abs_bits(z.y));
        if (lane == 0) {
          float worth;
          const float bound = __uint_as_float(left) + 2.f * __uint_as_float(grown);
          units[st][0] = unit_of(max(abs_bits(bound), abs_bits(inputs)), &worth);
          units[st][1] = worth;
          if (REV) units[st][2] = 128.f * fabsf(a.p.scale) * x * q * fac[st].last[1];
          mbar_arrive(smem_u32(&bars.unit_ready[st]));
        }
        __syncwarp();
      }
    }
  } else if (warp == kMmaWarp && (__syncwarp(), elect_one())) {
    // ---------------------------------------------------------------- products --
    auto wait = [&](uint64_t &b, uint32_t parity) { mbar_wait(smem_u32(&b), parity, a.p.status, &abort_flag); };
    const uint32_t id_k = idesc_f16(128, 64, BF, false, false), id_mn = idesc_f16(128, 64, BF, false, true);
    const uint32_t id_u = idesc_f16(128, D, BF, false, true);   // update: N = key channels
    const uint32_t id_a64 = idesc_f16(128, 64, BF, true, true);  // dO^T from shared memory
    while (step_piece(), take_piece()) {
      for (int pos = p0; pos < p1; ++pos, ++it) {
        const int st = it & 1;
        const uint32_t base = sb + st * L::kStage;
        const KMajor k_rows(base + L::K, 8192), q_rows(base + L::Q, 8192);
        const MNMajor k_cols(base + L::K, 8192), q_cols(base + L::Q, 8192);
        wait(bars.full[st], (it >> 1) & 1);
        if (pos == rp) wait_tail(st);
        // key channels in the order in which the chain hands them over: quarters 0 and 2, then 1 and 3
        wait(bars.s_ready[0], it & 1);
        tc_fence_after();
        constexpr int H4 = D / 32;  // steps of half the key channels
        issue_ts<0, 2>(tmem + cR1, tmem + cSH, k_rows, id_k, false);
        issue_ts<0, 2>(tmem + cR1, tmem + cSL, k_rows, id_k, true);
        issue_ts<H4, H4 + 2>(tmem + cR1, tmem + cSH, k_rows, id_k, true);
        issue_ts<H4, H4 + 2>(tmem + cR1, tmem + cSL, k_rows, id_k, true);
        if (D == 128) {
          wait(bars.s_ready[1], it & 1);
          tc_fence_after();
          issue_ts<2, 4>(tmem + cR1, tmem + cSH, k_rows, id_k, true);
          issue_ts<2, 4>(tmem + cR1, tmem + cSL, k_rows, id_k, true);
          issue_ts<6, 8>(tmem + cR1, tmem + cSH, k_rows, id_k, true);
          issue_ts<6, 8>(tmem + cR1, tmem + cSL, k_rows, id_k, true);
        }
        mma_commit(smem_u32(&bars.ks_done));
        if (MODE == kOut) {
          if (it > 0) wait(bars.out_free, (it - 1) & 1);
          tc_fence_after();
          issue_ts<0, D / 16>(tmem + cR2, tmem + cSH, q_rows, id_k, false);
          issue_ts<0, D / 16>(tmem + cR2, tmem + cSL, q_rows, id_k, true);
        }
        if (REV) {  // dO^T P T
          const MNMajor dO(base + L::V, 8192);
          issue_ss<0, 4>(tmem + cR2, dO, MNMajor(base + L::T + 8192, 0), id_a64, false);
          issue_ss<0, 4>(tmem + cR2, dO, MNMajor(base + L::T + 16384 + 8192, 0), id_a64, true);
        }
        wait(bars.x_ready, it & 1);
        tc_fence_after();
        if (REV) {
          const MNMajor th(base + L::T, 0), tl(base + L::T + 16384, 0);
          constexpr uint32_t at = BF ? cR2 : cR1;  // fp16: apart from dO's part, which is in another unit
          issue_ts<0, 4>(tmem + at, tmem + cXH, th, id_mn, BF);
          issue_ts<0, 4>(tmem + at, tmem + cXH, tl, id_mn, true);
          issue_ts<0, 4>(tmem + at, tmem + cXL, th, id_mn, true);
          mma_commit(smem_u32(&bars.u_done));
          wait(bars.qs_ready, it & 1);
          tc_fence_after();
          issue_ts<0, 4>(tmem + cS, tmem + cR3, q_cols, id_u, true);
          issue_ts<0, 4>(tmem + cS, tmem + cR3 + 32, q_cols, id_u, true);
        } else {
          const KMajor th(base + L::T, 0), tl(base + L::T + 16384, 0);
          issue_ts<0, 4>(tmem + cR1, tmem + cXH, th, id_k, false);
          issue_ts<0, 4>(tmem + cR1, tmem + cXH, tl, id_k, true);
          issue_ts<0, 4>(tmem + cR1, tmem + cXL, th, id_k, true);
          mma_commit(smem_u32(&bars.u_done));
        }
        if (MODE == kOut) {
          const KMajor ph(base + L::T + 8192, 0), pl(base + L::T + 16384 + 8192, 0);
          issue_ts<0, 4>(tmem + cR3, tmem + cXH, ph, id_k, false);
          issue_ts<0, 4>(tmem + cR3, tmem + cXH, pl, id_k, true);
          issue_ts<0, 4>(tmem + cR3, tmem + cXL, ph, id_k, true);
          mma_commit(smem_u32(&bars.o_done));
        }
        wait(bars.up_ready, it & 1);
        tc_fence_after();
        const uint32_t up = tmem + (MODE == kOut ? cSH : cXH);
        issue_ts<0, 4>(tmem + cS, up, k_cols, id_u, true);
        issue_ts<0, 4>(tmem + cS, up + 32, k_cols, id_u, true);
        mma_commit(smem_u32(&bars.s_done));
        mma_commit(smem_u32(&bars.empty[st]));
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMmaWarp) tmem_dealloc(tmem, 512);
}

template <int D, bool BF, int MODE>
__global__ void __launch_bounds__(kScanThreads<BF>, 1) scan_kernel(const __grid_constant__ Args a, const __grid_constant__ Maps maps) {
  scan_cta<D, BF, MODE>(a, maps, blockIdx.x);
}

// The backward's two scans side by side, where there are SMs for both: neither needs the other.  (On
// half of the SMs each where there are not, they took longer: 1210 against 1170 us for 16 x 2048 tokens' step.)
template <int D, bool BF>
__global__ void __launch_bounds__(kScanThreads<BF>, 1)
    scan_pair_kernel(const __grid_constant__ Args a, const __grid_constant__ Maps store, const __grid_constant__ Maps rev) {
  if (blockIdx.x < a.ranges)
    scan_cta<D, BF, kRev>(a, rev, blockIdx.x);
  else
    scan_cta<D, BF, kStore>(a, store, blockIdx.x - a.ranges);
}

template <int D>
constexpr uint32_t prep_smem() {
  constexpr uint32_t kq = 128 * D * 2, mat = 2 * 64 * kLd * 4;  // and 32 KB of two-term tiles
  return kq > mat ? kq : mat;
}

template <int D, bool BF>
bool make_maps(const Args &a, int mode, Maps *m) {
  const kda_delta_params &p = a.p;
  *m = {};
  if (a.max_chunks == 0 || p.T == 0) return true;
  auto view = [](const kda_tensor &t) { return View{t.data, t.stride_b, t.stride_h, t.stride_t, t.stride_d}; };
  const kda_tensor &v = mode == kRev ? p.dout : p.v, &o = mode == kRev ? p.dv : (mode == kOut ? p.o : p.v);
  return make_tmap_bhtd(&m->k, view(p.k), p.B, p.Hk, p.T, D, BF) && make_tmap_bhtd(&m->q, view(p.q), p.B, p.Hk, p.T, D, BF) &&
         make_tmap_bhtd(&m->v, view(v), p.B, p.H, p.T, D, BF) && make_tmap_bhtd(&m->o, view(o), p.B, p.H, p.T, D, BF);
}

template <int D, bool BF, int MODE>
cudaError_t run_scan(const Args &a, cudaStream_t st) {
  Maps m;
  if (!make_maps<D, BF>(a, MODE, &m)) return cudaErrorInvalidValue;
  constexpr uint32_t smem = ScanSmem<D, MODE>::kBytes;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(scan_kernel<D, BF, MODE>, smem, done);
  if (e != cudaSuccess) return e;
  e = launch_kernel(scan_kernel<D, BF, MODE>, dim3((unsigned)a.ranges), dim3(kScanThreads<BF>), smem, st, true, a, m);
  count_launches(1);
  return e;
}

template <int D, bool BF>
cudaError_t run_backward(const Args &a, cudaStream_t st) {
  if (2 * a.ranges > a.sms) {
    const cudaError_t e = run_scan<D, BF, kStore>(a, st);
    return e == cudaSuccess ? run_scan<D, BF, kRev>(a, st) : e;
  }
  Maps m1, m2;
  if (!make_maps<D, BF>(a, kStore, &m1) || !make_maps<D, BF>(a, kRev, &m2)) return cudaErrorInvalidValue;
  constexpr uint32_t smem = ScanSmem<D, kRev>::kBytes;
  static_assert(smem >= ScanSmem<D, kStore>::kBytes, "");
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(scan_pair_kernel<D, BF>, smem, done);
  if (e != cudaSuccess) return e;
  e = launch_kernel(scan_pair_kernel<D, BF>, dim3(2 * (unsigned)a.ranges), dim3(kScanThreads<BF>), smem, st, true, a, m1, m2);
  count_launches(1);
  return e;
}

template <int D, bool BF>
cudaError_t run_prep(const Args &a, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(prep_kernel<D, BF>, prep_smem<D>(), done);
  if (e != cudaSuccess) return e;
  e = launch_kernel(prep_kernel<D, BF>, dim3((unsigned)a.max_chunks, (unsigned)a.p.H), dim3(kPrepThreads), prep_smem<D>(), st,
                    a.p.cu_seqlens != nullptr, a);
  count_launches(1);
  return e;
}

}  // namespace

cudaError_t launch_plan(const Args &a, cudaStream_t st) {
  plan_kernel<<<1, 1024, 0, st>>>(a);
  count_launches(1);
  return cudaGetLastError();
}

#define KDA_DELTA_PICK(FN, ...)                                                                     \
  (a.p.dtype == KDA_DTYPE_BF16 ? (a.p.D == 64 ? FN<64, true __VA_ARGS__>(a, st) : FN<128, true __VA_ARGS__>(a, st)) \
                               : (a.p.D == 64 ? FN<64, false __VA_ARGS__>(a, st) : FN<128, false __VA_ARGS__>(a, st)))

cudaError_t launch_prep(const Args &a, cudaStream_t st) { return a.max_chunks == 0 ? cudaSuccess : KDA_DELTA_PICK(run_prep); }
cudaError_t launch_scan(const Args &a, cudaStream_t st) { return KDA_DELTA_PICK(run_scan, , kOut); }
cudaError_t launch_backward_scans(const Args &a, cudaStream_t st) { return KDA_DELTA_PICK(run_backward); }

}  // namespace delta
}  // namespace kda
