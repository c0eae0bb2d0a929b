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
// products a chunk: [K; Q] S, then [T; P T] X (or its transpose), then the state update,
// which accumulates on the state in tensor memory.  The columns of S are independent of
// one another, so a CTA carries 64 of them: 112 KB of shared memory and 256 columns of
// tensor memory, two CTAs an SM, which hide one another's waits.
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

// gamma and beta of a chunk, for one thread's row
struct Gates {
  float gi, gl, bi;
  __device__ __forceinline__ Gates(const Args &a, int chunk, int h, int row, bool live) : gi(0.f), gl(0.f), bi(0.f) {
    if (live) {
      const size_t at = ((size_t)chunk * a.p.H + h) * 64;
      gi = a.w.gam[at + row];
      gl = a.w.gam[at + 63];
      bi = a.w.beta[at + row];
    }
  }
};

template <int D>
struct ScanSmem {
  static constexpr uint32_t KQ = 0, T = KQ + 128 * D * 2, SH = T + kImgT, SL = SH + D * 128, B = SL + D * 128;
  static constexpr uint32_t kBytes = B + 16384;
};

// -------------------------------------------------------------- forward scan --
// One CTA per (sequence, head, 64 columns of the state).  STORE: instead of the outputs,
// the state before each chunk and the chunk's u rows go to the workspace (backward).
template <int D, bool BF, bool STORE>
__global__ void __launch_bounds__(kThreads, 2) scan_kernel(const Args a) {
  using L = ScanSmem<D>;
  constexpr int NS = D / 64;
  extern __shared__ __align__(1024) char smem[];
  __shared__ Ctl ctl;
  const int tid = threadIdx.x, sl = blockIdx.x % NS, h = blockIdx.x / NS % a.p.H, n = blockIdx.x / NS / a.p.H;
  if (n == a.nseq) {  // packed sequences: the rows outside them
    if (!STORE) zero_outside(a, a.p.o, h, 64 * sl);
    return;
  }
  const int hk = h / (a.p.H / a.p.Hk);
  const int row = tid & 127, half = tid >> 7, r64 = row & 63;
  const bool upper = row >= 64;  // warp-uniform: q rows (outputs); else k rows (u)
  const uint32_t sb = smem_u32(smem), lane_base = (uint32_t)((tid >> 5) & 3) << 21;
  const uint32_t tmem = cta_begin(ctl, 256);
  const uint32_t tS = tmem + lane_base + 32 * half, tR1 = tS + 64, tR2 = tS + 128;
  const Seq s = get_seq(a, n);
  const int nc = (s.len + kChunk - 1) / kChunk;
  const size_t st_off = (((size_t)n * a.p.H + h) * D + row) * D + 64 * sl + 32 * half;

  const uint16_t *kb = static_cast<const uint16_t *>(a.p.k.data) + s.b * a.p.k.stride_b + hk * a.p.k.stride_h + s.t0 * a.p.k.stride_t;
  const uint16_t *qb = static_cast<const uint16_t *>(a.p.q.data) + s.b * a.p.q.stride_b + hk * a.p.q.stride_h + s.t0 * a.p.q.stride_t;
  const uint16_t *vb = static_cast<const uint16_t *>(a.p.v.data) + s.b * a.p.v.stride_b + h * a.p.v.stride_h +
                       (s.t0 + r64) * a.p.v.stride_t + 64 * sl + 32 * half;
  uint16_t *ob = static_cast<uint16_t *>(a.p.o.data) + s.b * a.p.o.stride_b + h * a.p.o.stride_h +
                 (s.t0 + r64) * a.p.o.stride_t + 64 * sl + 32 * half;

  auto load_kq = [&](int c) {
    const int rows = min(kChunk, s.len - c * kChunk);
    load_rows<D>(sb + L::KQ, 0, 16384, kb + (int64_t)c * kChunk * a.p.k.stride_t, a.p.k.stride_t, rows);
    if (!STORE) load_rows<D>(sb + L::KQ, 64, 16384, qb + (int64_t)c * kChunk * a.p.q.stride_t, a.p.q.stride_t, rows);
  };
  auto load_t = [&](int c) {  // one thread
    mbar_arrive_expect_tx(smem_u32(&ctl.load_bar), kImgT);
    bulk_load(sb + L::T, a.w.T + ((size_t)(s.chunk0 + c) * a.p.H + h) * kImgT, kImgT, smem_u32(&ctl.load_bar));
  };

  uint32_t ph = 0, ph_load = 0;
  if (nc > 0) {
    load_kq(0);
    if (tid == 0) load_t(0);
  }
  float x[32];
  if (nc > 0 || a.p.state_out != nullptr) {
#pragma unroll
    for (int j = 0; j < 32; ++j) x[j] = 0.f;
    if (row < D && a.p.state_in != nullptr)
#pragma unroll
      for (int j = 0; j < 32; j += 4) *reinterpret_cast<float4 *>(x + j) = *reinterpret_cast<const float4 *>(a.p.state_in + st_off + j);
  }
  Gates gates(a, s.chunk0, h, r64, nc > 0);
  for (int c = 0; c < nc; ++c) {
    const int rows = min(kChunk, s.len - c * kChunk);
    const size_t ch = (size_t)(s.chunk0 + c) * a.p.H + h;
    const float gi = gates.gi, gl = gates.gl, bi = gates.bi;
    if (c + 1 < nc) {  // the next chunk: gates on their way, rows into L2
      const int next = min(kChunk, s.len - (c + 1) * kChunk);
      gates = Gates(a, s.chunk0 + c + 1, h, r64, true);
      prefetch_rows<D>(kb + (int64_t)(c + 1) * kChunk * a.p.k.stride_t, a.p.k.stride_t, next);
      if (!STORE) prefetch_rows<D>(qb + (int64_t)(c + 1) * kChunk * a.p.q.stride_t, a.p.q.stride_t, next);
      if (half == 0 && !upper && r64 < next)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(vb + (int64_t)(c + 1) * kChunk * a.p.v.stride_t));
    }
    uint4 vraw[4];
    if (!upper) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        vraw[j] = r64 < rows ? *reinterpret_cast<const uint4 *>(vb + (int64_t)c * kChunk * a.p.v.stride_t + 8 * j) : make_uint4(0, 0, 0, 0);
    }
    // the state as a two-term operand; what the update adds to is last * S
    if (row < D) {
      if (c > 0) tmem_ld32(tS, x);
      store_split32<BF>(sb + L::SH, sb + L::SL, row, half, x);
      if (STORE) {
        char *img = a.w.S + (ch * NS + sl) * (size_t)(D * 256);
        store_split32<BF>(img, img + D * 128, row, half, x);
      }
      const float last = exp_fast(gl);
#pragma unroll
      for (int j = 0; j < 32; ++j) x[j] *= last;
      tmem_st32(tS, x);
    }
    cp_async_wait();
    publish();
    if (tid == 0) {
      tc_fence_after();
      const uint32_t id = idesc_f16(128, 64, BF, false, true);
      issue<D / 16>(tmem + 64, KMajor{sb + L::KQ, 16384}, MNMajor{sb + L::SH, 0}, id, false);
      issue<D / 16>(tmem + 64, KMajor{sb + L::KQ, 16384}, MNMajor{sb + L::SL, 0}, id, true);
      mma_commit(smem_u32(&ctl.mma_bar));
    }
    wait_bar(ctl.mma_bar, ph, ctl, a.p.status);
    const float G = exp_fast(gi);
    tmem_ld32(tR1, x);
    if (!upper) {  // X = beta (V - G K S)
      float v[32];
#pragma unroll
      for (int j = 0; j < 4; ++j) unpack8<BF>(vraw[j], v + 8 * j);
#pragma unroll
      for (int j = 0; j < 32; ++j) x[j] = bi * fmaf(-G, x[j], v[j]);
      store_split32<BF>(sb + L::B, sb + L::B + 8192, r64, half, x);
    } else {
      const float f = a.p.scale * G;
#pragma unroll
      for (int j = 0; j < 32; ++j) x[j] *= f;
    }
    publish();
    if (tid == 0) {
      mbar_wait(smem_u32(&ctl.load_bar), ph_load, a.p.status, &ctl.abort);
      tc_fence_after();
      const uint32_t id = idesc_f16(128, 64, BF, false, true);
      const KMajor th{sb + L::T, 0}, tl{sb + L::T + 16384, 0};
      const MNMajor xh{sb + L::B, 0}, xl{sb + L::B + 8192, 0};
      issue<4>(tmem + 128, th, xh, id, false);
      issue<4>(tmem + 128, th, xl, id, true);
      issue<4>(tmem + 128, tl, xh, id, true);
      mma_commit(smem_u32(&ctl.mma_bar));
    }
    ph_load ^= 1;
    wait_bar(ctl.mma_bar, ph, ctl, a.p.status);
    if (tid == 0 && c + 1 < nc) load_t(c + 1);
    {
      float y[32];
      tmem_ld32(tR2, y);
      if (!upper) {
        if (STORE) {
          char *img = a.w.U + (ch * NS + sl) * (size_t)16384;
          store_split32<BF>(img, img + 8192, r64, half, y);
        }
        const float w = exp_fast(gl - gi);
#pragma unroll
        for (int j = 0; j < 32; ++j) y[j] *= w;
        store_split32<BF>(sb + L::B, sb + L::B + 8192, r64, half, y);
      } else if (!STORE && r64 < rows) {
#pragma unroll
        for (int j = 0; j < 32; ++j) x[j] += y[j];
        store_row32<BF>(ob + (int64_t)c * kChunk * a.p.o.stride_t, x);
      }
    }
    publish();
    if (tid == 0) {
      tc_fence_after();
      // D = 64: the second half of the 128 output rows reads other bytes of shared memory and is not used
      const uint32_t id = idesc_f16(128, 64, BF, true, true);
      const MNMajor kt{sb + L::KQ, 16384};
      issue<4>(tmem, kt, MNMajor{sb + L::B, 0}, id, true);
      issue<4>(tmem, kt, MNMajor{sb + L::B + 8192, 0}, id, true);
      mma_commit(smem_u32(&ctl.mma_bar));
    }
    wait_bar(ctl.mma_bar, ph, ctl, a.p.status);
    if (c + 1 < nc) load_kq(c + 1);
  }
  if (row < D && !STORE && a.p.state_out != nullptr) {
    if (nc > 0) tmem_ld32(tS, x);
#pragma unroll
    for (int j = 0; j < 32; j += 4) *reinterpret_cast<float4 *>(a.p.state_out + st_off + j) = *reinterpret_cast<float4 *>(x + j);
  }
  cta_end(tmem, 256);
}

// -------------------------------------------------------------- reverse scan --
// One CTA per (sequence, head, 64 columns of the state gradient), last chunk first.  Writes
// dV, the state gradient after each chunk and dX for the gradient kernel.
template <int D>
struct RevSmem {
  static constexpr uint32_t KQ = 0, T = KQ + 128 * D * 2, SH = T + kImgT, SL = SH + D * 128;
  // second operand tiles [128 x 64]; the lo tile takes the place of the state gradient's lo tile
  static constexpr uint32_t BL = SL, BH = SL + 16384;
  static constexpr uint32_t kBytes = BH + 16384;
};

template <int D, bool BF>
__global__ void __launch_bounds__(kThreads, 2) rev_kernel(const Args a) {
  using L = RevSmem<D>;
  constexpr int NS = D / 64;
  extern __shared__ __align__(1024) char smem[];
  __shared__ Ctl ctl;
  const int tid = threadIdx.x, sl = blockIdx.x % NS, h = blockIdx.x / NS % a.p.H, n = blockIdx.x / NS / a.p.H;
  const int G_ = a.p.H / a.p.Hk, hk = h / G_;
  if (n == a.nseq) {
    zero_outside(a, a.p.dv, h, 64 * sl);
    if (h % G_ == 0) {
      zero_outside(a, a.p.dq, hk, 64 * sl);
      zero_outside(a, a.p.dk, hk, 64 * sl);
    }
    if (sl == 0) {
      zero_outside(a, a.p.dg, a.p.g_dtype, h);
      zero_outside(a, a.p.dbeta, a.p.beta_dtype, h);
    }
    return;
  }
  const int row = tid & 127, half = tid >> 7, r64 = row & 63;
  const bool upper = row >= 64;
  const uint32_t sb = smem_u32(smem), lane_base = (uint32_t)((tid >> 5) & 3) << 21;
  const uint32_t tmem = cta_begin(ctl, 256);
  const uint32_t tS = tmem + lane_base + 32 * half, tR1 = tS + 64, tR2 = tS + 128;
  const Seq s = get_seq(a, n);
  const int nc = (s.len + kChunk - 1) / kChunk;
  const size_t st_off = (((size_t)n * a.p.H + h) * D + row) * D + 64 * sl + 32 * half;
  const uint16_t *kb = static_cast<const uint16_t *>(a.p.k.data) + s.b * a.p.k.stride_b + hk * a.p.k.stride_h + s.t0 * a.p.k.stride_t;
  const uint16_t *qb = static_cast<const uint16_t *>(a.p.q.data) + s.b * a.p.q.stride_b + hk * a.p.q.stride_h + s.t0 * a.p.q.stride_t;
  const uint16_t *db = static_cast<const uint16_t *>(a.p.dout.data) + s.b * a.p.dout.stride_b + h * a.p.dout.stride_h +
                       (s.t0 + r64) * a.p.dout.stride_t + 64 * sl + 32 * half;
  uint16_t *vb = static_cast<uint16_t *>(a.p.dv.data) + s.b * a.p.dv.stride_b + h * a.p.dv.stride_h +
                 (s.t0 + r64) * a.p.dv.stride_t + 64 * sl + 32 * half;
  auto load_kq = [&](int c) {
    const int rows = min(kChunk, s.len - c * kChunk);
    load_rows<D>(sb + L::KQ, 0, 16384, kb + (int64_t)c * kChunk * a.p.k.stride_t, a.p.k.stride_t, rows);
    load_rows<D>(sb + L::KQ, 64, 16384, qb + (int64_t)c * kChunk * a.p.q.stride_t, a.p.q.stride_t, rows);
  };
  auto load_t = [&](int c) {
    mbar_arrive_expect_tx(smem_u32(&ctl.load_bar), kImgT);
    bulk_load(sb + L::T, a.w.T + ((size_t)(s.chunk0 + c) * a.p.H + h) * kImgT, kImgT, smem_u32(&ctl.load_bar));
  };
  uint32_t ph = 0, ph_load = 0;
  if (nc > 0) {
    load_kq(nc - 1);
    if (tid == 0) load_t(nc - 1);
  }
  float x[32];
#pragma unroll
  for (int j = 0; j < 32; ++j) x[j] = 0.f;
  if (row < D && a.p.dstate_out != nullptr)
#pragma unroll
    for (int j = 0; j < 32; j += 4) *reinterpret_cast<float4 *>(x + j) = *reinterpret_cast<const float4 *>(a.p.dstate_out + st_off + j);
  Gates gates(a, s.chunk0 + nc - 1, h, r64, nc > 0);
  for (int c = nc - 1; c >= 0; --c) {
    const int rows = min(kChunk, s.len - c * kChunk);
    const size_t ch = (size_t)(s.chunk0 + c) * a.p.H + h;
    const float gi = gates.gi, gl = gates.gl, bi = gates.bi;
    if (c > 0) {  // the chunk before: gates on their way, rows into L2
      gates = Gates(a, s.chunk0 + c - 1, h, r64, true);
      prefetch_rows<D>(kb + (int64_t)(c - 1) * kChunk * a.p.k.stride_t, a.p.k.stride_t, kChunk);
      prefetch_rows<D>(qb + (int64_t)(c - 1) * kChunk * a.p.q.stride_t, a.p.q.stride_t, kChunk);
      if (half == 0 && upper)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(db + (int64_t)(c - 1) * kChunk * a.p.dout.stride_t));
    }
    uint4 draw[4];
    if (upper) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        draw[j] = r64 < rows ? *reinterpret_cast<const uint4 *>(db + (int64_t)c * kChunk * a.p.dout.stride_t + 8 * j) : make_uint4(0, 0, 0, 0);
    }
    if (row < D) {
      if (c < nc - 1) tmem_ld32(tS, x);
      store_split32<BF>(sb + L::SH, sb + L::SL, row, half, x);
      char *img = a.w.dS + (ch * NS + sl) * (size_t)(D * 256);
      store_split32<BF>(img, img + D * 128, row, half, x);
      const float last = exp_fast(gl);
#pragma unroll
      for (int j = 0; j < 32; ++j) x[j] *= last;
      tmem_st32(tS, x);
    }
    if (upper) {  // dO as it is: the second 64 rows of the [Z; dO] operand
#pragma unroll
      for (int j = 0; j < 4; ++j) sts(sb + L::BH + chunk_at(row, 4 * half + j), draw[j]);
    }
    cp_async_wait();
    publish();
    if (tid == 0) {
      tc_fence_after();
      const uint32_t id = idesc_f16(128, 64, BF, false, true);
      issue<D / 16>(tmem + 64, KMajor{sb + L::KQ, 16384}, MNMajor{sb + L::SH, 0}, id, false);
      issue<D / 16>(tmem + 64, KMajor{sb + L::KQ, 16384}, MNMajor{sb + L::SL, 0}, id, true);
      mma_commit(smem_u32(&ctl.mma_bar));
    }
    wait_bar(ctl.mma_bar, ph, ctl, a.p.status);
    if (!upper) {  // Z
      tmem_ld32(tR1, x);
      const float w = exp_fast(gl - gi);
#pragma unroll
      for (int j = 0; j < 32; ++j) x[j] *= w;
      store_split32<BF>(sb + L::BH, sb + L::BL, row, half, x);
    }
    publish();
    if (tid == 0) {
      mbar_wait(smem_u32(&ctl.load_bar), ph_load, a.p.status, &ctl.abort);
      tc_fence_after();
      // [T; P T]^T [Z; dO]: 64 output rows; the other 64 read other bytes of the image and are not used
      const uint32_t id = idesc_f16(128, 64, BF, true, true);
      const MNMajor th{sb + L::T, 16384}, tl{sb + L::T + 16384, 0};
      const MNMajor bh{sb + L::BH, 0}, bl{sb + L::BL, 0};
      issue<8>(tmem + 128, th, bh, id, false);
      issue<8>(tmem + 128, tl, bh, id, true);
      issue<4>(tmem + 128, th, bl, id, true);
      mma_commit(smem_u32(&ctl.mma_bar));
    }
    ph_load ^= 1;
    wait_bar(ctl.mma_bar, ph, ctl, a.p.status);
    if (tid == 0 && c > 0) load_t(c - 1);
    const float G = exp_fast(gi);
    if (!upper) {
      tmem_ld32(tR2, x);
      char *img = a.w.dX + (ch * NS + sl) * (size_t)16384;
      store_split32<BF>(img, img + 8192, r64, half, x);
#pragma unroll
      for (int j = 0; j < 32; ++j) x[j] *= bi;
      if (r64 < rows) store_row32<BF>(vb + (int64_t)c * kChunk * a.p.dv.stride_t, x);
#pragma unroll
      for (int j = 0; j < 32; ++j) x[j] *= -G;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) unpack8<BF>(draw[j], x + 8 * j);
      const float f = a.p.scale * G;
#pragma unroll
      for (int j = 0; j < 32; ++j) x[j] *= f;
    }
    store_split32<BF>(sb + L::BH, sb + L::BL, row, half, x);
    publish();
    if (tid == 0) {
      tc_fence_after();
      const uint32_t id = idesc_f16(128, 64, BF, true, true);
      const MNMajor kq{sb + L::KQ, 16384};
      issue<8>(tmem, kq, MNMajor{sb + L::BH, 0}, id, true);
      issue<8>(tmem, kq, MNMajor{sb + L::BL, 0}, id, true);
      mma_commit(smem_u32(&ctl.mma_bar));
    }
    wait_bar(ctl.mma_bar, ph, ctl, a.p.status);
    if (c > 0) load_kq(c - 1);
  }
  if (row < D && a.p.dstate_in != nullptr) {
    if (nc > 0) tmem_ld32(tS, x);
#pragma unroll
    for (int j = 0; j < 32; j += 4) *reinterpret_cast<float4 *>(a.p.dstate_in + st_off + j) = *reinterpret_cast<float4 *>(x + j);
  }
  cta_end(tmem, 256);
}

template <typename K>
cudaError_t run(K kern, dim3 grid, uint32_t smem, const Args &a, cudaStream_t st) {
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  kern<<<grid, kThreads, smem, st>>>(a);
  count_launches(1);
  return cudaGetLastError();
}

template <int D>
constexpr uint32_t prep_smem() {
  constexpr uint32_t kq = 128 * D * 2, mat = 2 * 64 * kLd * 4;
  return ((kq > mat ? kq : mat) + 1023) / 1024 * 1024 + kImgT;
}

unsigned scan_grid(const Args &a) {
  return (unsigned)((a.nseq + (a.p.cu_seqlens != nullptr ? 1 : 0)) * a.p.H * (a.p.D / 64));
}

}  // namespace

cudaError_t launch_plan(const Args &a, cudaStream_t st) {
  plan_kernel<<<1, 1024, 0, st>>>(a);
  count_launches(1);
  return cudaGetLastError();
}

#define KDA_DELTA_PICK(FN, SM, GRID)                                                       \
  do {                                                                                     \
    const bool bf = a.p.dtype == KDA_DTYPE_BF16;                                           \
    if (a.p.D == 64) return bf ? run(FN(64, true), GRID, SM(64), a, st) : run(FN(64, false), GRID, SM(64), a, st); \
    return bf ? run(FN(128, true), GRID, SM(128), a, st) : run(FN(128, false), GRID, SM(128), a, st);              \
  } while (0)

cudaError_t launch_prep(const Args &a, cudaStream_t st) {
  if (a.max_chunks == 0) return cudaSuccess;
  const dim3 grid((unsigned)a.max_chunks, (unsigned)a.p.H);
#define FN(D, BF) prep_kernel<D, BF>
#define SM(D) prep_smem<D>()
  KDA_DELTA_PICK(FN, SM, grid);
#undef FN
#undef SM
}

cudaError_t launch_scan(const Args &a, bool store, cudaStream_t st) {
#define SM(D) ScanSmem<D>::kBytes
  if (store) {
#define FN(D, BF) scan_kernel<D, BF, true>
    KDA_DELTA_PICK(FN, SM, dim3(scan_grid(a)));
#undef FN
  }
#define FN(D, BF) scan_kernel<D, BF, false>
  KDA_DELTA_PICK(FN, SM, dim3(scan_grid(a)));
#undef FN
#undef SM
}

cudaError_t launch_rev(const Args &a, cudaStream_t st) {
#define FN(D, BF) rev_kernel<D, BF>
#define SM(D) RevSmem<D>::kBytes
  KDA_DELTA_PICK(FN, SM, dim3(scan_grid(a)));
#undef FN
#undef SM
}

}  // namespace delta
}  // namespace kda
