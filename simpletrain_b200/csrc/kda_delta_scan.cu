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
#include "kda_delta_tc.cuh"

namespace kda {
namespace delta {
namespace {

// ------------------------------------------------------------ sequence plan --
// bound[i] = cu_seqlens[i] clamped into [0, T] and to no less than its predecessors;
// first[i] = chunks before sequence i.
__global__ void __launch_bounds__(1024) plan_kernel(const Args a) {
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

// One CTA per (chunk, head): T and P T as two-term images, gamma and beta in fp32.
// The products are k.k, q.k and P T; (I + A)^-1 is by halves in fp32: four 16 x 16 blocks
// by substitution, a column a thread, then [A 0; B C]^-1 = [a 0; -c B a, c] twice.
template <int D, bool BF>
__global__ void __launch_bounds__(kThreads) prep_kernel(const Args a) {
  constexpr uint32_t KQ = 0, kKQ = 128 * D * 2;
  constexpr uint32_t kMat = 2 * 64 * kLd * 4;
  constexpr uint32_t TT = ((kKQ > kMat ? kKQ : kMat) + 1023) / 1024 * 1024;  // [T; P] hi, then lo
  extern __shared__ __align__(1024) char smem[];
  __shared__ Ctl ctl;
  __shared__ __align__(16) float gam[64], bet[64];
  int64_t b, t0;
  int rows;
  if (!get_chunk(a, blockIdx.x, &b, &t0, &rows)) return;
  const int h = blockIdx.y, hk = h / (a.p.H / a.p.Hk), tid = threadIdx.x;
  const int row = tid & 127, half = tid >> 7, r64 = row & 63;
  const uint32_t sb = smem_u32(smem), lane_base = (uint32_t)((tid >> 5) & 3) << 21;
  load_rows<D>(sb + KQ, 0, 16384, static_cast<const uint16_t *>(a.p.k.data) + b * a.p.k.stride_b + hk * a.p.k.stride_h + t0 * a.p.k.stride_t,
               a.p.k.stride_t, rows);
  load_rows<D>(sb + KQ, 64, 16384, static_cast<const uint16_t *>(a.p.q.data) + b * a.p.q.stride_b + hk * a.p.q.stride_h + t0 * a.p.q.stride_t,
               a.p.q.stride_t, rows);
  const uint32_t tmem = cta_begin(ctl, 128);
  const size_t ch = (size_t)blockIdx.x * a.p.H + h;
  if (tid < 32) {
    // running sums in double: rounded once, so that differences of gammas keep fp32's last bits
    double s[2];
    for (int j = 0; j < 2; ++j) {
      const int i = 2 * tid + j;
      s[j] = i < rows ? (double)fmaxf(load_gate(a.p.g, b * a.p.g_stride_b + h * a.p.g_stride_h + (t0 + i) * a.p.g_stride_t, a.p.g_dtype), kMinGate) : 0.0;
      bet[i] = i < rows ? load_gate(a.p.beta, b * a.p.beta_stride_b + h * a.p.beta_stride_h + (t0 + i) * a.p.beta_stride_t, a.p.beta_dtype) : 0.f;
    }
    double c = s[0] + s[1];
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, c, o);
      if (tid >= o) c += y;
    }
    gam[2 * tid + 1] = (float)c;
    gam[2 * tid] = (float)(c - s[1]);
  }
  cp_async_wait();
  publish();
  uint32_t ph = 0;
  if (tid == 0) {
    tc_fence_after();
    issue<D / 16>(tmem, KMajor{sb + KQ, 16384}, KMajor{sb + KQ, 16384}, idesc_f16(128, 64, BF, false, false), false);
    mma_commit(smem_u32(&ctl.mma_bar));
  }
  if (tid < 64) {
    a.w.gam[ch * 64 + tid] = gam[tid];
    a.w.beta[ch * 64 + tid] = bet[tid];
  }
  const float gi = gam[r64] * kLog2e, bi = bet[r64];
  wait_bar(ctl.mma_bar, ph, ctl, a.p.status);
  float *As = reinterpret_cast<float *>(smem + KQ);  // over the k and q tiles: their product is done
  float *Ti = As + 64 * kLd;
  {
    float x[32];
    tmem_ld32(tmem + lane_base + 32 * half, x);
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      const int col = 32 * half + j;
      const float d = ex2f(fmaf(-kLog2e, gam[col], gi));
      if (row < 64)
        x[j] = col < r64 ? bi * d * x[j] : 0.f;
      else
        x[j] = col <= r64 ? a.p.scale * d * x[j] : 0.f;
    }
    if (row < 64) {
#pragma unroll
      for (int j = 0; j < 32; j += 4)
        *reinterpret_cast<float4 *>(As + r64 * kLd + 32 * half + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
    } else {
      store_split32<BF>(sb + TT, sb + TT + 16384, row, half, x);
    }
  }
  __syncthreads();
  if (tid < 64) {
    // column j of the inverse of diagonal block blk
    const int blk = tid >> 4, j = tid & 15, o = 16 * blk;
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s = i == j ? 1.f : 0.f;
#pragma unroll
      for (int m = 0; m < i; ++m) s = fmaf(-As[(o + i) * kLd + o + m], x[m], s);
      x[i] = i < j ? 0.f : s;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) Ti[(o + i) * kLd + o + j] = x[i];
  } else {
    // the blocks above the diagonal
    for (int e = tid - 64; e < 4096; e += kThreads - 64) {
      const int i = e >> 6, j = e & 63;
      if ((j >> 4) > (i >> 4)) Ti[i * kLd + j] = 0.f;
    }
  }
  __syncthreads();
#pragma unroll
  for (int n = 16; n < 64; n *= 2) {
    // for each pair of diagonal n-blocks: the block below them, -c B a, through the unused block of A above them
    const int pairs = 32 / n, per = n * n / 4, work = pairs * per;  // float4 outputs
    for (int e = tid; e < work; e += kThreads) {
      const int p = e / per, f = e % per, i = f / (n / 4), j = f % (n / 4) * 4, o = 2 * n * p;
      float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
      for (int m = 0; m < n; ++m) {
        const float l = As[(o + n + i) * kLd + o + m];
        const float4 r = *reinterpret_cast<const float4 *>(Ti + (o + m) * kLd + o + j);
        s.x = fmaf(l, r.x, s.x);
        s.y = fmaf(l, r.y, s.y);
        s.z = fmaf(l, r.z, s.z);
        s.w = fmaf(l, r.w, s.w);
      }
      *reinterpret_cast<float4 *>(As + (o + i) * kLd + o + n + j) = s;
    }
    __syncthreads();
    for (int e = tid; e < work; e += kThreads) {
      const int p = e / per, f = e % per, i = f / (n / 4), j = f % (n / 4) * 4, o = 2 * n * p;
      float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
      for (int m = 0; m < n; ++m) {
        const float l = Ti[(o + n + i) * kLd + o + n + m];
        const float4 r = *reinterpret_cast<const float4 *>(As + (o + m) * kLd + o + n + j);
        s.x = fmaf(-l, r.x, s.x);
        s.y = fmaf(-l, r.y, s.y);
        s.z = fmaf(-l, r.z, s.z);
        s.w = fmaf(-l, r.w, s.w);
      }
      *reinterpret_cast<float4 *>(Ti + (o + n + i) * kLd + o + j) = s;
    }
    __syncthreads();
  }
  if (row < 64) {
    float x[32];
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
      const float4 r = *reinterpret_cast<const float4 *>(Ti + r64 * kLd + 32 * half + j);
      x[j] = r.x;
      x[j + 1] = r.y;
      x[j + 2] = r.z;
      x[j + 3] = r.w;
    }
    store_split32<BF>(sb + TT, sb + TT + 16384, row, half, x);
  }
  publish();
  if (tid == 0) {
    tc_fence_after();
    // rows 64..127: P T (rows 0..63, T T, are not read)
    const uint32_t id = idesc_f16(128, 64, BF, false, true);
    const KMajor ph_{sb + TT, 0}, pl{sb + TT + 16384, 0};
    const MNMajor th{sb + TT, 0}, tl{sb + TT + 16384, 0};
    issue<4>(tmem + 64, ph_, th, id, false);
    issue<4>(tmem + 64, ph_, tl, id, true);
    issue<4>(tmem + 64, pl, th, id, true);
    mma_commit(smem_u32(&ctl.mma_bar));
  }
  wait_bar(ctl.mma_bar, ph, ctl, a.p.status);
  if (row >= 64) {
    float x[32];
    tmem_ld32(tmem + lane_base + 64 + 32 * half, x);
    store_split32<BF>(sb + TT, sb + TT + 16384, row, half, x);
  }
  fence_async_smem();
  cta_end(tmem, 128);
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
  for (int64_t e = threadIdx.x; e < rows * 8; e += kThreads) {
    const int64_t r = e >> 3, t = r < lo ? r : r - lo + hi;
    *reinterpret_cast<uint4 *>(base + t * o.stride_t + (e & 7) * 8) = make_uint4(0, 0, 0, 0);
  }
}
__device__ void zero_outside(const Args &a, void *p, int dtype, int h) {
  const int lo = a.w.bound[0], hi = a.w.bound[a.nseq];
  const int64_t rows = (int64_t)lo + (a.p.T - hi);
  for (int64_t r = threadIdx.x; r < rows; r += kThreads)
    store_gate(p, (int64_t)h * a.p.T + (r < lo ? r : r - lo + hi), dtype, 0.f);
}

// ------------------------------------------------------------------ the scans --
// One CTA per (sequence, head) and direction, with the state transposed in tensor memory:
// lanes are the value channels, columns the key channels, so that the operand that changes
// from step to step (the state, X, U) is always the first one and goes from registers
// straight back into tensor memory, split in two terms, without touching shared memory:
//   forward   [K S]^T = S^T K^T      X^T          U^T = X^T T^T          S^T += U'^T K
//   reverse   [K dS]^T = dS^T K^T    Z^T          dX^T = Z^T T + dO^T PT dS^T += dY^T K + dO^T Q'
// (U' = e^{gamma_63 - gamma} U, dY = -G beta dX, Q' = scale G Q).  A first version with the
// state as the second operand in shared memory spent 880 of 6750 cycles a chunk and half
// state on the first product alone: its operands, not its arithmetic, set the time.
//
// Warps: 8 walk the dependent chain (a value channel a thread, half the columns each), 4
// turn finished tiles into output or workspace rows, 3 load, one issues the products.
// Loads run one chunk ahead in two stages.
enum { kOut = 0, kStore = 1, kRev = 2 };  // outputs; state and u rows for the backward; reverse scan

constexpr int kScanThreads = 512;
constexpr int kOutWarp = 8, kLoadWarp = 12, kMmaWarp = 15;  // the chain: warps 0 .. 7
constexpr int kLoaders = 32 * (kMmaWarp - kLoadWarp);

// Per-token factors of a chunk, one array a factor: beta, -beta e^gamma, e^{gamma_63 - gamma}, scale e^gamma.
struct Factors {
  float beta[64], bg[64], w[64], sg[64];
  float last[4];  // e^{gamma_63}
};

template <int D, int MODE>
struct ScanSmem {
  static constexpr uint32_t KQ = 0, V = 128 * D * 2, T = V + 64 * D * 2, kStage = T + kImgT;
  static constexpr uint32_t OUT = 2 * kStage;  // outputs: [64 x D]; reverse: dX hi and lo
  static constexpr uint32_t kTile = 64 * D * 2;
  static constexpr uint32_t QS = OUT + 2 * kTile;  // reverse: Q' hi and lo
  static constexpr uint32_t kBytes = MODE == kOut ? OUT + kTile : (MODE == kRev ? QS + 2 * kTile : OUT);
};

struct ScanBars {
  uint64_t full[2], tfull[2], empty[2];
  uint64_t s_ready, ks_done, x_ready, u_done, up_ready, s_done, o_done, out_free, qs_ready;
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

// rows of a [T, D] view into D / 64 swizzled [64 x 64] blocks `block` bytes apart, by the loading threads
template <int D>
__device__ __forceinline__ void load_tile(uint32_t tile, uint32_t block, const uint16_t *base, int64_t stride_t, int rows,
                                             int t) {
  constexpr int P = D / 8;
#pragma unroll 4
  for (int p = t; p < 64 * P; p += kLoaders) {
    const int r = p / P, c = p % P;
    const bool live = r < rows;
    cp_async16(tile + (c >> 3) * block + r * 128 + (((c & 7) ^ (r & 7)) << 4), base + (live ? r * stride_t : 0) + c * 8, live);
  }
}

__device__ __forceinline__ void stmatrix_x4_trans(uint32_t addr, uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(r0), "r"(r1), "r"(r2),
               "r"(r3)
               : "memory");
}

template <int D, bool BF, int MODE>
__global__ void __launch_bounds__(kScanThreads, 1) scan_kernel(const Args a) {
  using L = ScanSmem<D, MODE>;
  constexpr int Q = D / 32;  // warps that own live tensor-memory lanes, of four
  constexpr bool REV = MODE == kRev;
  extern __shared__ __align__(1024) char smem[];
  __shared__ ScanBars bars;
  __shared__ __align__(16) Factors fac[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int h = blockIdx.x % a.p.H, n = blockIdx.x / a.p.H, G_ = a.p.H / a.p.Hk, hk = h / G_;
  if (n == a.nseq) {  // packed sequences: the rows outside them
    for (int c = 0; c < D; c += 64) {
      if (MODE == kOut) zero_outside(a, a.p.o, h, c);
      if (REV) {
        zero_outside(a, a.p.dv, h, c);
        if (h % G_ == 0) {
          zero_outside(a, a.p.dq, hk, c);
          zero_outside(a, a.p.dk, hk, c);
        }
      }
    }
    if (REV) {
      zero_outside(a, a.p.dg, a.p.g_dtype, h);
      zero_outside(a, a.p.dbeta, a.p.beta_dtype, h);
    }
    return;
  }
  const uint32_t sb = smem_u32(smem);
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&bars.full[i]), kLoaders);
      mbar_init(smem_u32(&bars.tfull[i]), 1);
      mbar_init(smem_u32(&bars.empty[i]), MODE == kStore ? 1 : 1 + Q);
    }
    for (uint64_t *b : {&bars.s_ready, &bars.x_ready, &bars.up_ready}) mbar_init(smem_u32(b), 2 * Q);
    for (uint64_t *b : {&bars.ks_done, &bars.u_done, &bars.s_done, &bars.o_done}) mbar_init(smem_u32(b), 1);
    mbar_init(smem_u32(&bars.out_free), Q);
    mbar_init(smem_u32(&bars.qs_ready), kLoaders);
    mbar_fence_init();
    abort_flag = 0;
  }
  if (warp == kMmaWarp) {
    tmem_alloc(smem_u32(&tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(&tmem_slot);
  auto wait = [&](uint64_t &b, uint32_t parity) { mbar_wait(smem_u32(&b), parity, a.p.status, &abort_flag); };
  auto arrive_warp = [&](uint64_t &b) {  // after this warp's tensor-memory accesses
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&b));
  };

  const Seq s = get_seq(a, n);
  const int nc = (s.len + kChunk - 1) / kChunk;
  auto chunk_of = [&](int it) { return REV ? nc - 1 - it : it; };
  auto cell = [&](int it) { return (size_t)(s.chunk0 + chunk_of(it)) * a.p.H + h; };

  if (warp < kOutWarp) {
    // ------------------------------------------------------------- the chain --
    const int quad = warp & 3, half = warp >> 2;
    if (quad < Q) {
      const uint32_t tl = tmem + ((uint32_t)quad << 21);
      const int dv = 32 * quad + lane;
      constexpr int W = D / 2;  // key channels of this thread
      const float *src = REV ? a.p.dstate_out : a.p.state_in;
      const size_t st_off = (((size_t)n * a.p.H + h) * D + half * W) * D + dv;
      // byte offsets of column dv in rows t = 0..7 of a swizzled tile
      uint32_t vcol[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) vcol[i] = (uint32_t)((dv >> 6) * 8192 + i * 128 + ((((dv >> 3) ^ i) & 7) << 4) + (dv & 7) * 2);
      for (int it = 0; it < nc; ++it) {
        const int st = it & 1;
        wait(bars.full[st], (it >> 1) & 1);
        const float last = fac[st].last[0];
        if (it > 0) {
          wait(bars.s_done, (it - 1) & 1);
          if (MODE != kOut) wait(bars.out_free, (it - 1) & 1);
        }
        __syncwarp();
        tc_fence_after();
#pragma unroll
        for (int c0 = 0; c0 < W; c0 += 32) {
          float x[32];
          if (it > 0) {
            tmem_ld32(tl + cS + half * W + c0, x);
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) x[j] = src != nullptr ? src[st_off + (size_t)(c0 + j) * D] : 0.f;
          }
          tmem_split32<BF>(tl + cSH + (half * W + c0) / 2, tl + cSL + (half * W + c0) / 2, x);
          uint32_t r[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(x[j] * last);
          tmem_st_32x32b_x32_nowait(tl + cS + half * W + c0, r);
        }
        tmem_wait_st();
        arrive_warp(bars.s_ready);
        float v[32];
        if (!REV) {  // V^T: this value channel of 32 tokens
          const uint32_t vt = sb + st * L::kStage + L::V + half * 4096;
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            uint16_t u;
            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(u) : "r"(vt + vcol[j & 7] + (j >> 3) * 1024));
            v[j] = unpack2((uint32_t)u, BF).x * fac[st].beta[32 * half + j];
          }
        }
        wait(bars.ks_done, it & 1);
        __syncwarp();
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
        wait(bars.u_done, it & 1);
        __syncwarp();
        tc_fence_after();
        {
          float x[32];
          tmem_ld32(tl + (REV ? cR2 : cR1) + 32 * half, x);
#pragma unroll
          for (int j = 0; j < 32; ++j) x[j] *= REV ? fac[st].bg[32 * half + j] : fac[st].w[32 * half + j];
          // over an operand whose products are done: S^T's (outputs: X^T may still be in use), else X^T's
          const uint32_t at = MODE == kOut ? cSH : cXH;
          tmem_split32<BF>(tl + at + 16 * half, tl + at + 32 + 16 * half, x);
          tmem_wait_st();
          arrive_warp(bars.up_ready);
        }
      }
      float *dst = REV ? a.p.dstate_in : (MODE == kOut ? a.p.state_out : nullptr);
      if (dst != nullptr) {
        if (nc > 0) wait(bars.s_done, (nc - 1) & 1);
        __syncwarp();
        tc_fence_after();
#pragma unroll
        for (int c0 = 0; c0 < W; c0 += 32) {
          float x[32];
          if (nc > 0) tmem_ld32(tl + cS + half * W + c0, x);
#pragma unroll
          for (int j = 0; j < 32; ++j)
            dst[st_off + (size_t)(c0 + j) * D] = nc > 0 ? x[j] : (src != nullptr ? src[st_off + (size_t)(c0 + j) * D] : 0.f);
        }
      }
    }
  } else if (warp < kLoadWarp) {
    // ------------------------------------------------------ finished tiles out --
    const int quad = warp & 3;
    if (quad < Q) {
      const uint32_t tl = tmem + ((uint32_t)quad << 21);
      const int t = tid - kOutWarp * 32;  // 0 .. 32 Q - 1
      const int mat = lane >> 3, rho = lane & 7;
      // address of the 16-byte run that this lane gives stmatrix for columns (tokens) 8 j .. 8 j + 15, lanes 16 hh ..
      auto st_at = [&](uint32_t tile, int hh, int j) {
        const int m0 = 32 * quad + 16 * hh + 8 * (mat & 1), tok = 8 * (j + (mat >> 1)) + rho;
        return tile + (uint32_t)((m0 >> 6) * 8192) + chunk_at(tok, (m0 & 63) >> 3);
      };
      for (int it = 0; it < nc; ++it) {
        const int st = it & 1, c = chunk_of(it), rows = min(kChunk, s.len - c * kChunk);
        if (MODE == kOut) {
          wait(bars.o_done, it & 1);
          __syncwarp();
          tc_fence_after();
          const int q2 = 2 * (lane & 3);
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            uint32_t qs[32], o[32];
            tmem_ld_16x256b_x8(tl + ((uint32_t)(16 * hh) << 16) + cR2, qs);
            tmem_ld_16x256b_x8(tl + ((uint32_t)(16 * hh) << 16) + cR3, o);
            uint32_t pk[16];  // [column block j][row half]
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float f0 = fac[st].sg[8 * j + q2], f1 = fac[st].sg[8 * j + q2 + 1];
#pragma unroll
              for (int e = 0; e < 2; ++e)
                pk[2 * j + e] = pack2(fmaf(f0, __uint_as_float(qs[4 * j + 2 * e]), __uint_as_float(o[4 * j + 2 * e])),
                                      fmaf(f1, __uint_as_float(qs[4 * j + 2 * e + 1]), __uint_as_float(o[4 * j + 2 * e + 1])), BF);
            }
#pragma unroll
            for (int j = 0; j < 8; j += 2)
              stmatrix_x4_trans(st_at(sb + L::OUT, hh, j), pk[2 * j], pk[2 * j + 1], pk[2 * j + 2], pk[2 * j + 3]);
          }
          arrive_warp(bars.out_free);
          if (lane == 0) mbar_arrive(smem_u32(&bars.empty[st]));
          named_bar_sync(1, 32 * Q);
          uint16_t *ob = static_cast<uint16_t *>(a.p.o.data) + s.b * a.p.o.stride_b + h * a.p.o.stride_h +
                         (s.t0 + (int64_t)c * kChunk) * a.p.o.stride_t;
#pragma unroll 4
          for (int e = t; e < 64 * (D / 8); e += 32 * Q) {
            const int r = e / (D / 8), g = e % (D / 8);
            if (r < rows)
              *reinterpret_cast<uint4 *>(ob + r * a.p.o.stride_t + 8 * g) = ld_shared_v4(sb + L::OUT + (g >> 3) * 8192 + chunk_at(r, g & 7));
          }
          named_bar_sync(1, 32 * Q);
        } else {
          // the state (reverse: its gradient) as the chain split it
          wait(bars.s_ready, it & 1);
          __syncwarp();
          tc_fence_after();
          char *img = (REV ? a.w.dS : a.w.S) + cell(it) * (size_t)(D * D * 4);
          const int row = 32 * quad + lane;
#pragma unroll
          for (int part = 0; part < 2; ++part)
#pragma unroll
            for (int b = 0; b < D / 64; ++b) {
              uint32_t r[32];
              tmem_ld_32x32b_x32(tl + (part ? cSL : cSH) + 32 * b, r);
              char *dst = img + part * (D * D * 2) + b * (D * 128);
#pragma unroll
              for (int g = 0; g < 8; ++g)
                *reinterpret_cast<uint4 *>(dst + chunk_at(row, g)) = make_uint4(r[4 * g], r[4 * g + 1], r[4 * g + 2], r[4 * g + 3]);
            }
          wait(bars.u_done, it & 1);
          __syncwarp();
          tc_fence_after();
          if (MODE == kStore) {  // U^T
            char *ui = a.w.U + cell(it) * (size_t)(D * 256);
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              float x[32];
              tmem_ld32(tl + cR1 + 32 * b, x);
              store_split32<BF>(ui, ui + D * 128, row, b, x);
            }
            arrive_warp(bars.out_free);
          } else {  // dX, and dV = beta dX
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
              uint32_t x[32], hi[16], lo[16];
              tmem_ld_16x256b_x8(tl + ((uint32_t)(16 * hh) << 16) + cR2, x);
#pragma unroll
              for (int i = 0; i < 16; ++i) split2<BF>(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1]), hi[i], lo[i]);
#pragma unroll
              for (int j = 0; j < 8; j += 2) {
                stmatrix_x4_trans(st_at(sb + L::OUT, hh, j), hi[2 * j], hi[2 * j + 1], hi[2 * j + 2], hi[2 * j + 3]);
                stmatrix_x4_trans(st_at(sb + L::OUT + L::kTile, hh, j), lo[2 * j], lo[2 * j + 1], lo[2 * j + 2], lo[2 * j + 3]);
              }
            }
            arrive_warp(bars.out_free);
            named_bar_sync(1, 32 * Q);
            char *xi = a.w.dX + cell(it) * (size_t)(D * 256);
            uint16_t *vb = static_cast<uint16_t *>(a.p.dv.data) + s.b * a.p.dv.stride_b + h * a.p.dv.stride_h +
                           (s.t0 + (int64_t)c * kChunk) * a.p.dv.stride_t;
#pragma unroll 2
            for (int e = t; e < 64 * (D / 8); e += 32 * Q) {
              const int r = e / (D / 8), g = e % (D / 8);
              const uint32_t off = chunk_at(r, g & 7);
              const uint4 xh = ld_shared_v4(sb + L::OUT + (g >> 3) * 8192 + off);
              const uint4 xl = ld_shared_v4(sb + L::OUT + L::kTile + (g >> 3) * 8192 + off);
              *reinterpret_cast<uint4 *>(xi + (g >> 3) * 16384 + off) = xh;
              *reinterpret_cast<uint4 *>(xi + (g >> 3) * 16384 + 8192 + off) = xl;
              if (r < rows) {
                const float be = fac[st].beta[r];
                float y[8], z[8];
                unpack8<BF>(xh, y);
                unpack8<BF>(xl, z);
#pragma unroll
                for (int j = 0; j < 8; ++j) y[j] = be * (y[j] + z[j]);
                *reinterpret_cast<uint4 *>(vb + r * a.p.dv.stride_t + 8 * g) =
                    make_uint4(pack2(y[0], y[1], BF), pack2(y[2], y[3], BF), pack2(y[4], y[5], BF), pack2(y[6], y[7], BF));
              }
            }
            named_bar_sync(1, 32 * Q);
            if (lane == 0) mbar_arrive(smem_u32(&bars.empty[st]));
          }
        }
      }
    }
  } else if (warp < kMmaWarp) {
    // ------------------------------------------------------------------ loads --
    const int t = tid - kLoadWarp * 32;
    const uint16_t *kb = static_cast<const uint16_t *>(a.p.k.data) + s.b * a.p.k.stride_b + hk * a.p.k.stride_h + s.t0 * a.p.k.stride_t;
    const uint16_t *qb = static_cast<const uint16_t *>(a.p.q.data) + s.b * a.p.q.stride_b + hk * a.p.q.stride_h + s.t0 * a.p.q.stride_t;
    const kda_tensor &vt = REV ? a.p.dout : a.p.v;
    const uint16_t *vb = static_cast<const uint16_t *>(vt.data) + s.b * vt.stride_b + h * vt.stride_h + s.t0 * vt.stride_t;
    auto load = [&](int it) {
      const int st = it & 1, c = chunk_of(it), rows = min(kChunk, s.len - c * kChunk);
      const int64_t r0 = (int64_t)c * kChunk;
      const uint32_t base = sb + st * L::kStage;
      if (it >= 2) wait(bars.empty[st], ((it >> 1) - 1) & 1);
      __syncwarp();
      load_tile<D>(base + L::KQ, 16384, kb + r0 * a.p.k.stride_t, a.p.k.stride_t, rows, t);
      if (MODE != kStore) load_tile<D>(base + L::KQ + 8192, 16384, qb + r0 * a.p.q.stride_t, a.p.q.stride_t, rows, t);
      load_tile<D>(base + L::V, 8192, vb + r0 * vt.stride_t, vt.stride_t, rows, t);
      asm volatile("cp.async.commit_group;" ::: "memory");
      if (t == 0) {
        mbar_arrive_expect_tx(smem_u32(&bars.tfull[st]), kImgT);
        bulk_load(base + L::T, a.w.T + cell(it) * kImgT, kImgT, smem_u32(&bars.tfull[st]));
      }
      if (t < 64) {
        const size_t at = cell(it) * 64;
        const float gi = a.w.gam[at + t], gl = a.w.gam[at + 63], be = a.w.beta[at + t], G = exp_fast(gi);
        fac[st].beta[t] = be;
        fac[st].bg[t] = -be * G;
        fac[st].w[t] = exp_fast(gl - gi);
        fac[st].sg[t] = a.p.scale * G;
        if (t == 0) fac[st].last[0] = exp_fast(gl);
      }
    };
    if (nc > 0) load(0);
    for (int it = 0; it < nc; ++it) {
      const int st = it & 1;
      asm volatile("cp.async.wait_all;" ::: "memory");
      fence_async_smem();
      mbar_arrive(smem_u32(&bars.full[st]));
      if (REV) {
        // Q' = scale e^gamma Q in two terms, once its last use (the previous chunk's update) is over
        if (it > 0) wait(bars.s_done, (it - 1) & 1);
        wait(bars.full[st], (it >> 1) & 1);
        __syncwarp();
#pragma unroll 4
        for (int e = t; e < 64 * (D / 8); e += kLoaders) {
          const int r = e / (D / 8), g = e % (D / 8);
          const uint32_t off = (g >> 3) * 8192 + chunk_at(r, g & 7);
          float x[8];
          unpack8<BF>(ld_shared_v4(sb + st * L::kStage + L::KQ + 8192 + (g >> 3) * 16384 + chunk_at(r, g & 7)), x);
          const float f = fac[st].sg[r];
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] *= f;
          uint4 hi, lo;
          split8<BF>(x, hi, lo);
          sts(sb + L::QS + off, hi);
          sts(sb + L::QS + L::kTile + off, lo);
        }
        fence_async_smem();
        mbar_arrive(smem_u32(&bars.qs_ready));
      }
      if (it + 1 < nc) load(it + 1);
    }
  } else if (lane == 0) {
    // ---------------------------------------------------------------- products --
    const uint32_t id_k = idesc_f16(128, 64, BF, false, false), id_mn = idesc_f16(128, 64, BF, false, true);
    const uint32_t id_u = idesc_f16(128, D, BF, false, true);          // update: N = key channels
    const uint32_t id_a64 = idesc_f16(128, 64, BF, true, true), id_aD = idesc_f16(128, D, BF, true, true);  // dO^T from shared memory
    for (int it = 0; it < nc; ++it) {
      const int st = it & 1;
      const uint32_t base = sb + st * L::kStage;
      wait(bars.full[st], (it >> 1) & 1);
      wait(bars.s_ready, it & 1);
      tc_fence_after();
      const KMajor k_rows(base + L::KQ, 16384), q_rows(base + L::KQ + 8192, 16384);
      const MNMajor k_cols(base + L::KQ, 16384);
      issue_ts<D / 16>(tmem + cR1, tmem + cSH, k_rows, id_k, false);
      issue_ts<D / 16>(tmem + cR1, tmem + cSL, k_rows, id_k, true);
      mma_commit(smem_u32(&bars.ks_done));
      if (MODE == kOut) {
        if (it > 0) wait(bars.out_free, (it - 1) & 1);
        tc_fence_after();
        issue_ts<D / 16>(tmem + cR2, tmem + cSH, q_rows, id_k, false);
        issue_ts<D / 16>(tmem + cR2, tmem + cSL, q_rows, id_k, true);
      }
      wait(bars.tfull[st], (it >> 1) & 1);
      if (REV) {
        // dO^T [64 value channels a block] against P T and Q'
        const MNMajor dO(base + L::V, 8192);
        issue<4>(tmem + cR2, dO, MNMajor(base + L::T + 8192, 0), id_a64, false);
        issue<4>(tmem + cR2, dO, MNMajor(base + L::T + 16384 + 8192, 0), id_a64, true);
        wait(bars.qs_ready, it & 1);
        tc_fence_after();
        issue<4>(tmem + cS, dO, MNMajor(sb + L::QS, 8192), id_aD, true);
        issue<4>(tmem + cS, dO, MNMajor(sb + L::QS + L::kTile, 8192), id_aD, true);
      }
      wait(bars.x_ready, it & 1);
      tc_fence_after();
      if (REV) {
        const MNMajor th(base + L::T, 0), tl(base + L::T + 16384, 0);
        issue_ts<4>(tmem + cR2, tmem + cXH, th, id_mn, true);
        issue_ts<4>(tmem + cR2, tmem + cXH, tl, id_mn, true);
        issue_ts<4>(tmem + cR2, tmem + cXL, th, id_mn, true);
      } else {
        const KMajor th(base + L::T, 0), tl(base + L::T + 16384, 0);
        issue_ts<4>(tmem + cR1, tmem + cXH, th, id_k, false);
        issue_ts<4>(tmem + cR1, tmem + cXH, tl, id_k, true);
        issue_ts<4>(tmem + cR1, tmem + cXL, th, id_k, true);
      }
      mma_commit(smem_u32(&bars.u_done));
      if (MODE == kOut) {
        const KMajor ph(base + L::T + 8192, 0), pl(base + L::T + 16384 + 8192, 0);
        issue_ts<4>(tmem + cR3, tmem + cXH, ph, id_k, false);
        issue_ts<4>(tmem + cR3, tmem + cXH, pl, id_k, true);
        issue_ts<4>(tmem + cR3, tmem + cXL, ph, id_k, true);
        mma_commit(smem_u32(&bars.o_done));
      }
      wait(bars.up_ready, it & 1);
      tc_fence_after();
      const uint32_t up = tmem + (MODE == kOut ? cSH : cXH);
      issue_ts<4>(tmem + cS, up, k_cols, id_u, true);
      issue_ts<4>(tmem + cS, up + 32, k_cols, id_u, true);
      mma_commit(smem_u32(&bars.s_done));
      mma_commit(smem_u32(&bars.empty[st]));
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMmaWarp) tmem_dealloc(tmem, 512);
}

template <typename K>
cudaError_t run(K kern, dim3 grid, int threads, uint32_t smem, const Args &a, cudaStream_t st) {
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  kern<<<grid, threads, smem, st>>>(a);
  count_launches(1);
  return cudaGetLastError();
}

template <int D>
constexpr uint32_t prep_smem() {
  constexpr uint32_t kq = 128 * D * 2, mat = 2 * 64 * kLd * 4;
  return ((kq > mat ? kq : mat) + 1023) / 1024 * 1024 + kImgT;
}

template <int D, bool BF>
cudaError_t run_scan(const Args &a, int mode, cudaStream_t st) {
  const dim3 grid((unsigned)((a.nseq + (a.p.cu_seqlens != nullptr ? 1 : 0)) * a.p.H));
  if (mode == kOut) return run(scan_kernel<D, BF, kOut>, grid, kScanThreads, ScanSmem<D, kOut>::kBytes, a, st);
  if (mode == kStore) return run(scan_kernel<D, BF, kStore>, grid, kScanThreads, ScanSmem<D, kStore>::kBytes, a, st);
  return run(scan_kernel<D, BF, kRev>, grid, kScanThreads, ScanSmem<D, kRev>::kBytes, a, st);
}

cudaError_t scan(const Args &a, int mode, cudaStream_t st) {
  const bool bf = a.p.dtype == KDA_DTYPE_BF16;
  if (a.p.D == 64) return bf ? run_scan<64, true>(a, mode, st) : run_scan<64, false>(a, mode, st);
  return bf ? run_scan<128, true>(a, mode, st) : run_scan<128, false>(a, mode, st);
}

}  // namespace

cudaError_t launch_plan(const Args &a, cudaStream_t st) {
  plan_kernel<<<1, 1024, 0, st>>>(a);
  count_launches(1);
  return cudaGetLastError();
}

cudaError_t launch_prep(const Args &a, cudaStream_t st) {
  if (a.max_chunks == 0) return cudaSuccess;
  const dim3 grid((unsigned)a.max_chunks, (unsigned)a.p.H);
  const bool bf = a.p.dtype == KDA_DTYPE_BF16;
  if (a.p.D == 64) return bf ? run(prep_kernel<64, true>, grid, kThreads, prep_smem<64>(), a, st)
                             : run(prep_kernel<64, false>, grid, kThreads, prep_smem<64>(), a, st);
  return bf ? run(prep_kernel<128, true>, grid, kThreads, prep_smem<128>(), a, st)
            : run(prep_kernel<128, false>, grid, kThreads, prep_smem<128>(), a, st);
}

cudaError_t launch_scan(const Args &a, bool store, cudaStream_t st) { return scan(a, store ? kStore : kOut, st); }
cudaError_t launch_rev(const Args &a, cudaStream_t st) { return scan(a, kRev, st); }

}  // namespace delta
}  // namespace kda
