// The gated delta rule's gradients of q, k, g and beta, chunk by chunk, and its C-ABI
// entry points.
//
// Mathematics, for one chunk and head with the state S before it, the gradient dS of the
// state after it, U = T X, dX (the reverse scan's), e_ij = e^{gamma_i - gamma_j},
// w_i = e^{gamma_63 - gamma_i}, G_i = e^{gamma_i}:
//   M_ij = -(dX U^T)_ij beta_i e_ij (i > j)      (gradient of k_i.k_j)
//   N_ij = scale (dO U^T)_ij e_ij (i >= j)       (gradient of q_i.k_j)
//   dQ = N K + scale G (dO S^T)
//   dK = M K + M^T K + N^T Q - G beta (dX S^T) + w (U dS^T)
//   dbeta_i = dX_i.v_i - G_i t_i - sum_j (dX U^T)_ij e_ij k_i.k_j,   t_i = k_i.(dX S^T)_i
// The gradient of gamma_i, row by row, is what those terms give through their e^gamma
// factors; with y_i = w_i k_i.(U dS^T)_i and Z_ij = M_ij k_i.k_j + N_ij q_i.k_j (i > j),
//   dgamma_i = scale G_i q_i.(dO S^T)_i - G_i beta_i t_i + sum_j Z_ij - sum_j Z_ji
//   dg_t = sum_{i >= t} dgamma_i + sum_{j < t} y_j + e^{gamma_63} <S, dS>
// (the y_j enter dgamma_j with a minus and dgamma_63 with a plus; they do not cancel summed this way).  Z's
// sums are taken of its elements and not from the rows of the products: those hold the diagonal's N_ii q_i.k_i in
// both, which has no decay, and what is left of it after the difference was 5e-7 whatever dg is (7% of it at g = -12).
//
// A CTA takes (chunk, query/key head) cells in turn, walks the value heads that share the
// head and sums their dq and dk in registers, in order: no atomics, the result does not
// depend on the launch.  The tiles of one value head fill an SM's shared memory, so the
// next head's are brought into L2 meanwhile; 16 warps, a token row and a quarter of the
// columns a thread, work off the products.
//
// Measured: 466 us for 16 x 2048 tokens, 10 heads of 128 (5120 cells of 288 KB: 3.3 TB/s, 26,000
// cycles a cell).  One value head's tiles are all that fit, so copies, products and what the threads make of them
// follow one another; what can overlap does (prefetch into L2, terms through the state under
// the second products).  Holding k and q rows in registers to free room for the next tiles spilled (514 us).
// In fp16, where M and N wait for their unit, 569 us.  Z's column sums, 18 shuffles a thread, are 16 us of it; all sixteen
// columns at once took registers that are not there (478 us).
#include "kda_delta_tc.cuh"

namespace kda {
namespace delta {
namespace {

constexpr int kGradThreads = 512;
// Products and copies are issued by warps whose threads own q rows: they have less to do with the results.
constexpr int kMmaWarp = 2, kCopyThread = 96;

template <int D>
struct GradSmem {
  static constexpr uint32_t kTile = 128 * D * 2;
  static constexpr uint32_t KQ = 0, AH = KQ + kTile, AL = AH + kTile;  // [dX; dO] hi, lo (dO's lo rows: zeros)
  static constexpr uint32_t U = AL + kTile, S = U + 256 * D;           // U^T: hi, lo
  static constexpr uint32_t DH = S + 4 * D * D;                        // S^T hi, lo, then dS^T lo over S^T lo; dS^T hi
  static constexpr uint32_t kBytes = DH + 2 * D * D;
  static constexpr uint32_t MN = AH;                                   // [M; N] hi, lo (D = 64: runs over AL)
};

__device__ __forceinline__ void prefetch_l2(const void *p, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(reinterpret_cast<uint64_t>(p)), "r"(bytes) : "memory");
}

// N consecutive fp32 columns of this warp's lanes
template <int N>
__device__ __forceinline__ void tmem_ldn(uint32_t taddr, float (&x)[N]) {
  static_assert(N == 16 || N == 32, "");
  if constexpr (N == 32) {
    tmem_ld32(taddr, x);
  } else {
    uint32_t r[16];
    tmem_ld_32x32b_x16(taddr, r);
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = __uint_as_float(r[i]);
  }
}

template <int D, bool BF>
__global__ void __launch_bounds__(kGradThreads, 1) grad_kernel(const Args a) {
  using L = GradSmem<D>;
  constexpr int NS = D / 64, W = D / 4;  // W: columns of a D-wide row that a thread owns
  constexpr uint32_t tG1 = 0, tG2 = 64, tG5 = 128, tG6 = 256, tG3 = 0, tG4 = 384;
  extern __shared__ __align__(1024) char smem[];
  __shared__ Ctl ctl;
  __shared__ uint64_t bar_g2, bar_s, bar_d;
  __shared__ __align__(16) float gam[128];  // hi, then lo
  __shared__ float sm_dot[16], sm_xv[64];
  __shared__ __align__(16) uint32_t sm_size[16];
  __shared__ volatile float sm_unit[2];
  __shared__ float sm_f[2][64], sm_t[2][64], sm_y[2][64], sm_r[2][64];  // [half of the columns][row]
  const int tid = threadIdx.x, row = tid & 127, part = tid >> 7, r64 = row & 63;
  const bool upper = row >= 64;
  const int G_ = a.p.H / a.p.Hk, cells = a.max_chunks * a.p.Hk;
  const uint32_t sb = smem_u32(smem), lane_base = (uint32_t)((tid >> 5) & 3) << 21;
  if (tid == 0) {
    mbar_init(smem_u32(&bar_g2), 1);
    mbar_init(smem_u32(&bar_s), 1);
    mbar_init(smem_u32(&bar_d), 1);
  }
  const uint32_t tmem = cta_begin(ctl, 512);
  const uint32_t lane_t = tmem + lane_base;
  uint32_t ph = 0;  // every barrier completes once a value head (bar_g2 twice)
  // this thread's W columns of its row of a [128 x D] tile, eight at a time
  auto own_chunk = [&](int c) { return ((part * W + 8 * c) >> 6) * 16384 + chunk_at(row, ((part * W) >> 3) + c); };
  auto rows_at = [](const kda_tensor &x, int64_t b, int64_t hd, int64_t t) {
    return static_cast<uint16_t *>(x.data) + b * x.stride_b + hd * x.stride_h + t * x.stride_t;
  };
  auto mma_leader = [&]() { return (tid >> 5) == kMmaWarp && elect_one(); };
  // the tiles of value head h of chunk cell cidx, all but k and q
  auto load_head = [&](int cidx, int h, int64_t b, int64_t t0, int rows) {
    const size_t ch = (size_t)cidx * a.p.H + h;
    if (tid == kCopyThread) {
      const uint32_t b1 = smem_u32(&ctl.load_bar), b2 = smem_u32(&bar_s);
      mbar_arrive_expect_tx(b1, NS * 16384 + D * 256);
      for (int s = 0; s < NS; ++s) {
        const char *x = a.w.dX + (ch * NS + s) * (size_t)16384;
        bulk_load(sb + L::AH + s * 16384, x, 8192, b1);
        bulk_load(sb + L::AL + s * 16384, x + 8192, 8192, b1);
      }
      bulk_load(sb + L::U, a.w.U + ch * (size_t)(D * 256), D * 256, b1);
      mbar_arrive_expect_tx(b2, D * D * 6);
      bulk_load(sb + L::S, a.w.S + ch * (size_t)(D * D * 4), D * D * 4, b2);
      bulk_load(sb + L::DH, a.w.dS + ch * (size_t)(D * D * 4), D * D * 2, b2);
    }
    load_rows<D, kGradThreads>(sb + L::AH, 64, rows_at(a.p.dout, b, h, t0), a.p.dout.stride_t, rows);
    if (upper)
#pragma unroll
      for (int c = 0; c < W / 8; ++c) sts(sb + L::AL + own_chunk(c), make_uint4(0, 0, 0, 0));
  };

  pdl_wait();
  int64_t b = 0, t0 = 0;
  int rows = 0, u = blockIdx.x;
  bool live = u < cells && get_chunk(a, u / a.p.Hk, &b, &t0, &rows);
  if (live) load_head(u / a.p.Hk, (u % a.p.Hk) * G_, b, t0, rows);
  while (live) {
    const int cidx = u / a.p.Hk, hk = u % a.p.Hk;
    load_rows<D, kGradThreads>(sb + L::KQ, 0, rows_at(a.p.k, b, hk, t0), a.p.k.stride_t, rows);
    load_rows<D, kGradThreads>(sb + L::KQ, 64, rows_at(a.p.q, b, hk, t0), a.p.q.stride_t, rows);
    float acc[W];
#pragma unroll
    for (int j = 0; j < W; ++j) acc[j] = 0.f;
    // the cell after this one
    const int un = u + (int)gridDim.x;
    int64_t nb = 0, nt = 0;
    int nrows = 0;
    const bool more = un < cells && get_chunk(a, un / a.p.Hk, &nb, &nt, &nrows);

    for (int hh = 0; hh < G_; ++hh) {
      const int h = hk * G_ + hh;
      const size_t ch = (size_t)cidx * a.p.H + h;
      const bool last = hh + 1 == G_;
      const float *gsrc = a.w.gam + ch * 128;
      if (tid < 128) gam[tid] = gsrc[tid];
      const float bi = a.w.beta[ch * 64 + r64];
      // fp16: what a unit of the S and U images (F), of the dS and dX images (R), and of this row's products with the
      // former is worth; read again where they are used, registers being what this kernel has least of
      if (!BF && tid < 2) sm_unit[tid] = a.w.unit[ch * kUnits + kUnitF + tid];
      auto worth_F = [&]() { return sm_unit[0]; };
      auto worth_R = [&]() { return sm_unit[1]; };
      auto worth_row = [&]() { return upper ? sm_unit[0] : sm_unit[0] * sm_unit[1]; };
      // two 16-byte runs of a row of V, eight threads a row
      constexpr int VR = D / 64;
      const int vr = tid >> 3, vc = tid & 7;
      uint4 vraw[VR];
#pragma unroll
      for (int c = 0; c < VR; ++c)
        vraw[c] = vr < rows ? *reinterpret_cast<const uint4 *>(rows_at(a.p.v, b, h, t0 + vr) + 8 * (vc + 8 * c)) : make_uint4(0, 0, 0, 0);
      cp_async_wait();
      publish();
      if (mma_leader()) {
        mbar_wait(smem_u32(&ctl.load_bar), ph, a.p.status, &ctl.abort);
        tc_fence_after();
        const uint32_t id64 = idesc_f16(128, 64, BF, false, false), id64t = idesc_f16(128, 64, BF, false, true);
        const uint32_t idD = idesc_f16(128, D, BF, false, true), id6 = idesc_f16(128, D, BF, true, true);
        issue<D / 16>(tmem + tG1, KMajor{sb + L::KQ, 16384}, KMajor{sb + L::KQ, 16384}, id64, false);
        const KMajor ah{sb + L::AH, 16384}, al{sb + L::AL, 16384};
        const MNPlain uh{sb + L::U, D}, ul{sb + L::U + D * 128, D};
        issue<D / 16>(tmem + tG2, ah, uh, id64t, false);
        issue<D / 16>(tmem + tG2, ah, ul, id64t, true);
        issue<D / 16>(tmem + tG2, al, uh, id64t, true);
        mma_commit(smem_u32(&bar_g2));
        mbar_wait(smem_u32(&bar_s), ph, a.p.status, &ctl.abort);
        tc_fence_after();
        const MNPlain sh{sb + L::S, D}, sl{sb + L::S + D * D * 2, D}, dh{sb + L::DH, D};
        issue<D / 16>(tmem + tG5, ah, sh, idD, false);
        issue<D / 16>(tmem + tG5, ah, sl, idD, true);
        issue<D / 16>(tmem + tG5, al, sh, idD, true);
        // 64 rows (tokens); the other 64 read bytes behind and are not used
        issue<D / 16>(tmem + tG6, uh, dh, id6, false);
        issue<D / 16>(tmem + tG6, ul, dh, id6, true);
        mma_commit(smem_u32(&ctl.mma_bar));
      }
      __syncwarp();
      {  // rows that come next, a 128-byte line a thread: k, q, dout, v
        const int64_t pb = last ? nb : b, pt = last ? nt : t0;
        const int nk = last ? un % a.p.Hk : hk, nh = last ? nk * G_ : h + 1, pr = last ? (more ? nrows : 0) : rows;
        const kda_tensor &x = part == 0 ? a.p.k : (part == 1 ? a.p.q : (part == 2 ? a.p.dout : a.p.v));
        const int r = row / (D / 64), c = row % (D / 64);
        if (r < pr && (last || part > 1))
          asm volatile("prefetch.global.L2 [%0];" ::"l"(rows_at(x, pb, part < 2 ? nk : nh, pt + r) + c * 64));
      }
      // dX . v, and the products of the two images, place by place
      mbar_wait(smem_u32(&ctl.load_bar), ph, a.p.status, &ctl.abort);
      float xv = 0.f;
#pragma unroll
      for (int c = 0; c < VR; ++c) {
        const uint32_t at = c * 16384 + chunk_at(vr, vc);
        float x[8], y[8], v[8];
        unpack8<BF>(ld_shared_v4(sb + L::AH + at), x);
        unpack8<BF>(ld_shared_v4(sb + L::AL + at), y);
        unpack8<BF>(vraw[c], v);
#pragma unroll
        for (int j = 0; j < 8; ++j) xv = fmaf(x[j] + y[j], v[j], xv);
      }
      for (int o = 4; o > 0; o >>= 1) xv += __shfl_xor_sync(0xffffffffu, xv, o);
      if (vc == 0) sm_xv[vr] = BF ? xv : xv * worth_R();
      mbar_wait(smem_u32(&bar_s), ph, a.p.status, &ctl.abort);
      // <S, dS> = <S, dS hi> now, <S hi, dS lo> when that has come (S lo . dS lo is below fp32's last bits)
      float dot = 0.f;
#pragma unroll
      for (int e = tid; e < D * D / 8; e += kGradThreads) {
        const uint32_t off = e * 16;
        float x[8], y[8];
        unpack8<BF>(ld_shared_v4(sb + L::S + off), x);
        unpack8<BF>(ld_shared_v4(sb + L::S + off + D * D * 2), y);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] += y[j];
        unpack8<BF>(ld_shared_v4(sb + L::DH + off), y);
#pragma unroll
        for (int j = 0; j < 8; ++j) dot = fmaf(x[j], y[j], dot);
      }
      // M, N (16 columns)
      mbar_wait(smem_u32(&bar_g2), 0, a.p.status, &ctl.abort);
      __syncwarp();
      tc_fence_after();
      uint4 mh[2], ml[2];
      float mn[BF ? 1 : 2][8];  // fp16: M, N until their unit is known
      uint32_t size = 0;
      const float y_unit = BF ? 1.f : worth_row();
      float held[2];   // Z's column sums over this warp's rows: the even warps' go to sm_f, then the odd ones'
      float rs = 0.f;  // k rows: sum_j (dX U^T)_ij e_ij k_i.k_j, with a minus; q rows: Z's part
      {
        const float gh = gam[r64], gl = gam[64 + r64];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t xr[8], yr[8];
          tmem_ld_32x32b_x8_nowait(lane_t + tG1 + 16 * part + 8 * c, xr);
          tmem_ld_32x32b_x8_nowait(lane_t + tG2 + 16 * part + 8 * c, yr);
          tmem_wait_ld_bind(xr, yr);
          float m8[8], z[8];
#pragma unroll
          for (int j4 = 0; j4 < 8; j4 += 4) {
            const float4 ch4 = *reinterpret_cast<const float4 *>(gam + 16 * part + 8 * c + j4);
            const float4 cl4 = *reinterpret_cast<const float4 *>(gam + 64 + 16 * part + 8 * c + j4);
            const float hi[4] = {ch4.x, ch4.y, ch4.z, ch4.w}, lo[4] = {cl4.x, cl4.y, cl4.z, cl4.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int j = j4 + i, col = 16 * part + 8 * c + j;
              const float e = decay(gh, gl, hi[i], lo[i]), y = BF ? __uint_as_float(yr[j]) : __uint_as_float(yr[j]) * y_unit;
              if (!upper) {
                const float m = col < r64 ? -y * e : 0.f;
                rs = col < r64 ? fmaf(m, __uint_as_float(xr[j]), rs) : rs;
                m8[j] = m * bi;
                z[j] = m8[j] * __uint_as_float(xr[j]);
              } else {
                m8[j] = col <= r64 ? a.p.scale * y * e : 0.f;
                z[j] = col < r64 ? m8[j] * __uint_as_float(xr[j]) : 0.f;
                rs += z[j];
              }
            }
          }
          {  // eight columns over the warp's 32 rows: half of them go to the other half of the lanes, three times over
            const int lane = tid & 31;
#pragma unroll
            for (int n = 4; n > 0; n >>= 1) {
              const bool hi = lane & (4 * n);
#pragma unroll
              for (int j = 0; j < n; ++j) {
                const float keep = hi ? z[j + n] : z[j], give = hi ? z[j] : z[j + n];
                z[j] = keep + __shfl_xor_sync(0xffffffffu, give, 4 * n);
              }
            }
            z[0] += __shfl_xor_sync(0xffffffffu, z[0], 2);
            z[0] += __shfl_xor_sync(0xffffffffu, z[0], 1);
            if ((row & 32) == 0 && (lane & 3) == 0) sm_f[row >> 6][16 * part + 8 * c + (lane >> 2)] = -z[0];
            held[c] = z[0];
          }
          if constexpr (BF) {
            split8<BF>(m8, mh[c], ml[c]);
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              mn[c][j] = m8[j];
              size = max(size, abs_bits(m8[j]));
            }
          }
        }
        if constexpr (!BF) {
          size = __reduce_max_sync(0xffffffffu, size);
          if ((tid & 31) == 0) sm_size[tid >> 5] = size;
        }
      }
      // over the dX / dO tiles once their products are done and every thread is past its reads of them and of S
      mbar_wait(smem_u32(&ctl.mma_bar), ph, a.p.status, &ctl.abort);
      __syncwarp();
      tc_fence_after();
      publish();
      if (tid == kCopyThread) {
        mbar_arrive_expect_tx(smem_u32(&bar_d), D * D * 2);
        bulk_load(sb + L::S + D * D * 2, a.w.dS + ch * (size_t)(D * D * 4) + D * D * 2, D * D * 2, smem_u32(&bar_d));
        // what the next value head loads comes into L2 behind that (one bulk request each: line by line through
        // the load/store units it held up everything else for 5000 cycles)
        if (!last || more) {
          const size_t nx = last ? (size_t)(un / a.p.Hk) * a.p.H + (un % a.p.Hk) * G_ : ch + 1;
          prefetch_l2(a.w.dX + nx * (size_t)(D * 256), D * 256);
          prefetch_l2(a.w.U + nx * (size_t)(D * 256), D * 256);
          prefetch_l2(a.w.S + nx * (size_t)(D * D * 4), D * D * 4);
          prefetch_l2(a.w.dS + nx * (size_t)(D * D * 4), D * D * 4);
        }
      }
      if ((row & 32) && (tid & 3) == 0)
#pragma unroll
        for (int c = 0; c < 2; ++c) sm_f[row >> 6][16 * part + 8 * c + ((tid & 31) >> 2)] -= held[c];
      float iMN = 1.f;
      if constexpr (!BF) {
        size = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint4 z = *reinterpret_cast<const uint4 *>(sm_size + 4 * w);
          size = max(size, max(max(z.x, z.y), max(z.z, z.w)));
        }
        const float sMN = unit_of(size, &iMN);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int j = 0; j < 8; ++j) mn[c][j] *= sMN;
          split8<BF>(mn[c], mh[c], ml[c]);
        }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        sts(sb + L::MN + chunk_at(row, 2 * part + c), mh[c]);
        sts(sb + L::MN + 16384 + chunk_at(row, 2 * part + c), ml[c]);
      }
      publish();
      if (mma_leader()) {
        tc_fence_after();
        const uint32_t id3 = idesc_f16(128, D, BF, false, true), id4 = idesc_f16(128, D, BF, true, true);
        const MNMajor kq{sb + L::KQ, 16384};
        issue<4>(tmem + tG3, KMajor{sb + L::MN, 0}, kq, id3, false);
        issue<4>(tmem + tG3, KMajor{sb + L::MN + 16384, 0}, kq, id3, true);
        // 64 rows (k tokens); the other 64 are not used
        issue<8>(tmem + tG4, MNMajor{sb + L::MN, 16384}, kq, id4, false);
        issue<8>(tmem + tG4, MNMajor{sb + L::MN + 16384, 16384}, kq, id4, true);
        mbar_wait(smem_u32(&bar_d), ph, a.p.status, &ctl.abort);
        tc_fence_after();
        issue<D / 16>(tmem + tG6, MNPlain{sb + L::U, D}, MNPlain{sb + L::S + D * D * 2, D}, idesc_f16(128, D, BF, true, true), true);
        mma_commit(smem_u32(&bar_g2));
      }
      __syncwarp();
      // meanwhile the terms through the state
      float f_dot = 0.f, t_dot = 0.f, y_dot = 0.f;
      {
        float x[W];
        tmem_ldn<W>(lane_t + tG5 + part * W, x);
        float f = ex2f(gam[r64]) * (upper ? a.p.scale : -bi);
        if constexpr (!BF) f *= worth_row();
#pragma unroll
        for (int c = 0; c < W / 8; ++c) {
          float k[8];
          unpack8<BF>(ld_shared_v4(sb + L::KQ + own_chunk(c)), k);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            t_dot = fmaf(k[j], x[8 * c + j], t_dot);
            acc[8 * c + j] = fmaf(f, x[8 * c + j], acc[8 * c + j]);
          }
        }
        f_dot = f * t_dot + (upper ? rs : bi * rs);
        if constexpr (!BF) t_dot *= worth_row();
      }
      mbar_wait(smem_u32(&bar_d), ph, a.p.status, &ctl.abort);
#pragma unroll
      for (int e = tid; e < D * D / 8; e += kGradThreads) {
        float x[8], y[8];
        unpack8<BF>(ld_shared_v4(sb + L::S + e * 16), x);
        unpack8<BF>(ld_shared_v4(sb + L::S + D * D * 2 + e * 16), y);
#pragma unroll
        for (int j = 0; j < 8; ++j) dot = fmaf(x[j], y[j], dot);
      }
      for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
      if ((tid & 31) == 0) sm_dot[tid >> 5] = dot;
      mbar_wait(smem_u32(&bar_g2), 1, a.p.status, &ctl.abort);
      __syncwarp();
      tc_fence_after();
      publish();
      // all products and reads of the tiles are done, k and q aside: the next value head's come in
      if (!last)
        load_head(cidx, h + 1, b, t0, rows);
      else if (more)
        load_head(un / a.p.Hk, (un % a.p.Hk) * G_, nb, nt, nrows);
      float wi = decay(gam[63], gam[127], gam[r64], gam[64 + r64]);
      if constexpr (!BF) wi *= worth_F() * worth_R();
#pragma unroll
      for (int c0 = 0; c0 < W; c0 += 16) {
        float x[16], y[16], z[16];
        tmem_ldn<16>(lane_t + tG3 + part * W + c0, x);
        if (!upper) {
          tmem_ldn<16>(lane_t + tG4 + part * W + c0, y);
          tmem_ldn<16>(lane_t + tG6 + part * W + c0, z);
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float k[8];
          unpack8<BF>(ld_shared_v4(sb + L::KQ + own_chunk(c0 / 8 + c)), k);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int i = 8 * c + j;
            if constexpr (!BF) {
              const float s = upper ? x[i] : x[i] + y[i], v = upper ? 0.f : wi * z[i];
              y_dot = fmaf(k[j], v, y_dot);
              acc[c0 + i] += fmaf(iMN, s, v);
            } else if (upper) {
              acc[c0 + i] += x[i];
            } else {
              const float v = wi * z[i];
              y_dot = fmaf(k[j], v, y_dot);
              acc[c0 + i] += (x[i] + y[i]) + v;
            }
          }
        }
      }
      // the rows' sums, in a fixed order: the quarters of k rows, then those of q rows
      for (int turn = 0; turn < 2; ++turn) {
        if (!upper && (part >> 1) == turn) {
          const int p = part & 1;
          const float z = 0.f;
          sm_f[p][r64] += f_dot;
          sm_t[p][r64] = (turn ? sm_t[p][r64] : z) + t_dot;
          sm_y[p][r64] = (turn ? sm_y[p][r64] : z) + y_dot;
          sm_r[p][r64] = (turn ? sm_r[p][r64] : z) + rs;
        }
        __syncthreads();
      }
      for (int turn = 0; turn < 2; ++turn) {
        if (upper && (part >> 1) == turn) sm_f[part & 1][r64] += f_dot;
        if (turn) tc_fence_before();
        __syncthreads();
      }
      tc_fence_after();
      if (tid < 32) {
        float f[2], y[2];
        float sd = 0.f;
        for (int w = 0; w < 16; ++w) sd += sm_dot[w];
        sd *= ex2f(gam[63]);
        if constexpr (!BF) sd *= worth_F() * worth_R();
        for (int j = 0; j < 2; ++j) {
          const int i = 2 * tid + j;
          f[j] = sm_f[0][i] + sm_f[1][i];
          y[j] = sm_y[0][i] + sm_y[1][i];
          if (i < rows)
            store_gate(a.p.dbeta, (b * a.p.H + h) * a.p.T + t0 + i, a.p.beta_dtype,
                       sm_xv[i] - ex2f(gam[i]) * (sm_t[0][i] + sm_t[1][i]) + (sm_r[0][i] + sm_r[1][i]));
        }
        // suffix sums of f, exclusive prefix sums of y
        float sf = f[0] + f[1], py = y[0] + y[1];
        for (int o = 1; o < 32; o <<= 1) {
          const float un_ = __shfl_down_sync(0xffffffffu, sf, o), v = __shfl_up_sync(0xffffffffu, py, o);
          if (tid + o < 32) sf += un_;
          if (tid >= o) py += v;
        }
        const float next = __shfl_down_sync(0xffffffffu, sf, 1), prev = __shfl_up_sync(0xffffffffu, py, 1);
        const float s1 = f[1] + (tid < 31 ? next : 0.f), p0 = tid > 0 ? prev : 0.f;
        if (2 * tid < rows) store_gate(a.p.dg, (b * a.p.H + h) * a.p.T + t0 + 2 * tid, a.p.g_dtype, (f[0] + s1) + p0 + sd);
        if (2 * tid + 1 < rows)
          store_gate(a.p.dg, (b * a.p.H + h) * a.p.T + t0 + 2 * tid + 1, a.p.g_dtype, s1 + (p0 + y[0]) + sd);
      }
      ph ^= 1;
      if (!last) __syncthreads();
    }
    // dk over k's tile, dq over q's, then out in whole rows
#pragma unroll
    for (int c = 0; c < W / 8; ++c)
      sts(sb + L::KQ + own_chunk(c), make_uint4(pack2(acc[8 * c], acc[8 * c + 1], BF), pack2(acc[8 * c + 2], acc[8 * c + 3], BF),
                                                pack2(acc[8 * c + 4], acc[8 * c + 5], BF), pack2(acc[8 * c + 6], acc[8 * c + 7], BF)));
    __syncthreads();
    {
      constexpr int P = D / 8;
      uint16_t *dk = rows_at(a.p.dk, b, hk, t0), *dq = rows_at(a.p.dq, b, hk, t0);
#pragma unroll
      for (int e = tid; e < 128 * P; e += kGradThreads) {
        const int r = e / P, c = e % P, rr = r & 63;
        if (rr < rows)
          *reinterpret_cast<uint4 *>((r < 64 ? dk + rr * a.p.dk.stride_t : dq + rr * a.p.dq.stride_t) + 8 * c) =
              ld_shared_v4(sb + L::KQ + (c >> 3) * 16384 + chunk_at(r, c & 7));
      }
    }
    __syncthreads();
    u = un;
    live = more;
    b = nb;
    t0 = nt;
    rows = nrows;
  }
  cta_end(tmem, 512);
}

template <int D, bool BF>
cudaError_t run_grad(const Args &a, cudaStream_t st) {
  constexpr uint32_t smem = GradSmem<D>::kBytes;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(grad_kernel<D, BF>, smem, done);
  if (e != cudaSuccess) return e;
  const int sms = a.sms;
  const int64_t cells = (int64_t)a.max_chunks * a.p.Hk;
  e = launch_kernel(grad_kernel<D, BF>, dim3((unsigned)(cells < sms ? cells : sms)), dim3(kGradThreads), smem, st, true, a);
  count_launches(1);
  return e;
}

}  // namespace

cudaError_t launch_grad(const Args &a, cudaStream_t st) {
  if (a.max_chunks == 0) return cudaSuccess;
  const bool bf = a.p.dtype == KDA_DTYPE_BF16;
  if (a.p.D == 64) return bf ? run_grad<64, true>(a, st) : run_grad<64, false>(a, st);
  return bf ? run_grad<128, true>(a, st) : run_grad<128, false>(a, st);
}

}  // namespace delta
}  // namespace kda

// ------------------------------------------------------------------- C ABI --
namespace {

using kda::delta::Args;

bool gate_ok(int32_t d) { return d == KDA_DTYPE_BF16 || d == KDA_DTYPE_F16 || d == KDA_DTYPE_F32; }

// Most chunks of a packed row: one more than the whole ones for each sequence that has a token.
int packed_chunks(const kda_delta_params *p) { return p->T / 64 + (p->nseq < p->T ? p->nseq : p->T); }

int check_sizes(const kda_delta_params *p) {
  if (p == nullptr) return KDA_ERR_NULL_ARGUMENT;
  if (p->B < 0 || p->H < 0 || p->Hk < 0 || p->T < 0) return KDA_ERR_BAD_SHAPE;
  if (p->D != 64 && p->D != 128) return KDA_ERR_UNSUPPORTED;
  if (p->dtype != KDA_DTYPE_BF16 && p->dtype != KDA_DTYPE_F16) return KDA_ERR_UNSUPPORTED;
  if (!gate_ok(p->g_dtype) || !gate_ok(p->beta_dtype)) return KDA_ERR_UNSUPPORTED;
  if (p->B > 0 && p->H > 0 && (p->Hk == 0 || p->H % p->Hk)) return KDA_ERR_BAD_SHAPE;
  if (p->cu_seqlens != nullptr && (p->B != 1 || p->nseq < 0)) return KDA_ERR_BAD_SHAPE;
  // a work range waits for a long sequence's state, and waits are bounded: 2^18 chunks are 0.6 to 0.9 s of 2
  if (p->cu_seqlens != nullptr && p->T > 1 << 24) return KDA_ERR_BAD_SHAPE;
  if (p->H > 65535) return KDA_ERR_BAD_SHAPE;  // a grid dimension
  const int64_t nseq = p->cu_seqlens != nullptr ? (int64_t)p->nseq + 1 : p->B;
  if (nseq * p->H * 2 > 0x7fffffff) return KDA_ERR_BAD_SHAPE;
  const int64_t chunks = p->cu_seqlens != nullptr ? packed_chunks(p) : (int64_t)p->B * (((int64_t)p->T + 63) / 64);
  if (chunks * p->H > 0x3fffffff) return KDA_ERR_BAD_SHAPE;
  return KDA_OK;
}

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

int sm_count() {
  static std::atomic<int> cache[64];  // by device; 0 = not asked yet
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return sms;
  const int known = cache[dev].load(std::memory_order_relaxed);
  if (known > 0) return known;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0) sms = 148;
  cache[dev].store(sms, std::memory_order_relaxed);
  return sms;
}

// CTAs of a scan: one an SM, and no more than there are streams (sequence, head).
int scan_ranges(int64_t nseq, int64_t H, int sms) {
  const int64_t n = nseq * H;
  return (int)(n < 1 ? 1 : (n < sms ? n : sms));
}

// Sizes and workspace regions; returns the bytes needed (p->workspace may be NULL).
size_t lay_out(const kda_delta_params *p, bool backward, Args *a) {
  a->p = *p;
  const bool packed = p->cu_seqlens != nullptr;
  a->nseq = packed ? p->nseq : p->B;
  a->per_seq = packed ? 0 : (int)(((int64_t)p->T + 63) / 64);
  a->max_chunks = packed ? packed_chunks(p) : p->B * a->per_seq;
  const size_t cells = (size_t)a->max_chunks * p->H;
  char *base = static_cast<char *>(p->workspace);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    char *r = base == nullptr ? nullptr : base + at;
    at += align256(bytes);
    return r;
  };
  a->w = {};
  if (packed) {
    a->w.bound = reinterpret_cast<int *>(take(4 * ((size_t)p->nseq + 1)));
    a->w.first = reinterpret_cast<int *>(take(4 * ((size_t)p->nseq + 1)));
  }
  a->sms = sm_count();
  a->ranges = scan_ranges(a->nseq, p->H, a->sms);
  a->w.queue = reinterpret_cast<int *>(take(sizeof(int) * 2 * ((size_t)a->ranges + 2)));
  a->w.slots = reinterpret_cast<float *>(take((backward ? 2 : 1) * ((size_t)a->ranges + 1) * p->D * p->D * 4));
  if (p->dtype == KDA_DTYPE_F16) a->w.cuts = reinterpret_cast<float2 *>(take((backward ? 2 : 1) * ((size_t)a->ranges + 1) * 8 * sizeof(float2)));
  a->w.gam = reinterpret_cast<float *>(take(cells * 512));
  a->w.beta = reinterpret_cast<float *>(take(cells * 256));
  if (p->dtype == KDA_DTYPE_F16) a->w.unit = reinterpret_cast<float *>(take(cells * kda::delta::kUnits * 4));
  a->w.T = take(cells * kda::delta::kImgT);
  if (backward) {
    a->w.S = take(cells * p->D * p->D * 4);
    a->w.dS = take(cells * p->D * p->D * 4);
    a->w.U = take(cells * p->D * 256);
    a->w.dX = take(cells * p->D * 256);
  }
  return at;
}

int check_view(const kda_tensor &t, int64_t B, int64_t H, int64_t T) {
  if (t.data == nullptr) return KDA_ERR_NULL_ARGUMENT;
  if (t.stride_d != 1 || (reinterpret_cast<uintptr_t>(t.data) & 15u)) return KDA_ERR_BAD_LAYOUT;
  if ((t.stride_b % 8) || (t.stride_h % 8) || (t.stride_t % 8)) return KDA_ERR_BAD_LAYOUT;
  // a dimension that is stepped over has a stride (TMA maps have no broadcast)
  if ((B > 1 && t.stride_b <= 0) || (H > 1 && t.stride_h <= 0) || (T > 1 && t.stride_t <= 0)) return KDA_ERR_BAD_LAYOUT;
  return KDA_OK;
}

bool misaligned(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

int check_common(const kda_delta_params *p, bool tokens) {
  if (tokens) {
    for (const kda_tensor *t : {&p->q, &p->k})
      if (const int rc = check_view(*t, p->B, p->Hk, p->T)) return rc;
    if (const int rc = check_view(p->v, p->B, p->H, p->T)) return rc;
    if (p->g == nullptr || p->beta == nullptr) return KDA_ERR_NULL_ARGUMENT;
  }
  if (misaligned(p->state_in)) return KDA_ERR_BAD_LAYOUT;
  return KDA_OK;
}

}  // namespace

extern "C" {

size_t kda_delta_fwd_workspace_bytes(const kda_delta_params *p) {
  Args a;
  if (check_sizes(p) != KDA_OK) return 0;
  return lay_out(p, false, &a);
}

size_t kda_delta_bwd_workspace_bytes(const kda_delta_params *p) {
  Args a;
  if (check_sizes(p) != KDA_OK) return 0;
  return lay_out(p, true, &a);
}

int kda_delta_fwd_sm100(const kda_delta_params *p, kda_stream_t stream) {
  int rc = check_sizes(p);
  if (rc != KDA_OK) return rc;
  if (p->B == 0 || p->H == 0) return KDA_OK;
  const bool tokens = p->T > 0;
  if ((rc = check_common(p, tokens)) != KDA_OK) return rc;
  if (tokens && (rc = check_view(p->o, p->B, p->H, p->T)) != KDA_OK) return rc;
  if (misaligned(p->state_out)) return KDA_ERR_BAD_LAYOUT;
  Args a;
  const size_t need = lay_out(p, false, &a);
  if (need > 0 && (p->workspace == nullptr || p->workspace_bytes < need || (reinterpret_cast<uintptr_t>(p->workspace) & 255u)))
    return KDA_ERR_WORKSPACE;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e = p->cu_seqlens != nullptr ? kda::delta::launch_plan(a, st) : cudaSuccess;
  if (e == cudaSuccess) e = kda::delta::launch_prep(a, st);
  if (e == cudaSuccess) e = kda::delta::launch_scan(a, st);
  return e == cudaSuccess ? KDA_OK : KDA_ERR_CUDA;
}

int kda_delta_bwd_sm100(const kda_delta_params *p, kda_stream_t stream) {
  int rc = check_sizes(p);
  if (rc != KDA_OK) return rc;
  if (p->B == 0 || p->H == 0) return KDA_OK;
  const bool tokens = p->T > 0;
  if ((rc = check_common(p, tokens)) != KDA_OK) return rc;
  if (tokens) {
    for (const kda_tensor *t : {&p->dout, &p->dv})
      if ((rc = check_view(*t, p->B, p->H, p->T)) != KDA_OK) return rc;
    for (const kda_tensor *t : {&p->dq, &p->dk})
      if ((rc = check_view(*t, p->B, p->Hk, p->T)) != KDA_OK) return rc;
    if (p->dg == nullptr || p->dbeta == nullptr) return KDA_ERR_NULL_ARGUMENT;
  }
  if (misaligned(p->dstate_out) || misaligned(p->dstate_in)) return KDA_ERR_BAD_LAYOUT;
  Args a;
  const size_t need = lay_out(p, true, &a);
  if (need > 0 && (p->workspace == nullptr || p->workspace_bytes < need || (reinterpret_cast<uintptr_t>(p->workspace) & 255u)))
    return KDA_ERR_WORKSPACE;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e = p->cu_seqlens != nullptr ? kda::delta::launch_plan(a, st) : cudaSuccess;
  if (e == cudaSuccess) e = kda::delta::launch_prep(a, st);
  if (e == cudaSuccess) e = kda::delta::launch_backward_scans(a, st);
  if (e == cudaSuccess) e = kda::delta::launch_grad(a, st);
  return e == cudaSuccess ? KDA_OK : KDA_ERR_CUDA;
}

}  // extern "C"
