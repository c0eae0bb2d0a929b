// torch dispatcher ops over the C ABIs of include/kda_sm100.h and
// include/st_fused_ops.h:
//   kda_b200::chunk_fwd / chunk_bwd            -> kda_fwd_sm100 / kda_bwd_sm100
//   kda_b200::delta_fwd / delta_bwd            -> kda_delta_fwd_sm100 / kda_delta_bwd_sm100
//   kda_b200::delta_step                       -> kda_delta_step_sm100
//   st_b200::silu_mul / silu_mul_bwd           -> st_silu_mul_fwd / _bwd
//   st_b200::rmsnorm_residual / _bwd           -> st_rmsnorm_residual_fwd / _bwd
//   st_b200::cross_entropy / cross_entropy_bwd -> st_cross_entropy_fwd / _bwd
//   st_b200::token_logprobs / _bwd             -> st_token_logprobs_fwd / _bwd
//
// The schemas and CUDA implementations live here, in C++, so a call costs a
// dispatcher hop and a few caching-allocator allocations instead of a Python
// function; fake (meta) implementations and, but for the delta rule and the
// token log probabilities, autograd are registered from Python
// (simpletrain_b200/ops.py).  Those two have their autograd here: behind a
// Python formula a small training step cost 130 us of host time.  Outputs and the workspace come from the
// caching allocator and the kernels run on the current stream, so the ops can
// be captured in CUDA graphs.  Layout rules follow the ABI: a tensor whose
// innermost stride is not 1, whose other strides are not multiples of 8
// elements, or whose base is not 16-byte aligned is made contiguous first.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <cstdint>
#include <mutex>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/kda_sm100.h"
#include "../../include/st_fused_ops.h"

namespace {

using at::Tensor;
using c10::optional;

bool abi_layout_ok(const Tensor &t) {
  if (t.stride(-1) != 1 && t.size(-1) != 1) return false;
  if (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) return false;
  for (int64_t i = 0; i + 1 < t.dim(); ++i)
    if (t.size(i) != 1 && (t.stride(i) % 8 || t.stride(i) == 0)) return false;  // a broadcast dimension has no TMA map
  return true;
}

// (a copy of a contiguous tensor whose base is misaligned: contiguous() would hand it back)
Tensor prep(const Tensor &t) { return abi_layout_ok(t) ? t : t.clone(at::MemoryFormat::Contiguous); }

// New [B, H, T, D] tensor in the dimension order of `like`: its strides when
// they are dense, else [B, T, H, D] memory when `like` is time-major (the KDA
// layer's projection views, models/kimi_k3.py:99-102, dense or not), else
// contiguous.  Keeps the layer's transpose + contiguous() after the scan free.
Tensor empty_in_order_of(const Tensor &like) {
  if (like.is_non_overlapping_and_dense()) return at::empty_like(like);
  if (like.stride(1) < like.stride(2))
    return at::empty({like.size(0), like.size(2), like.size(1), like.size(3)}, like.options()).transpose(1, 2);
  return at::empty(like.sizes(), like.options());
}

optional<Tensor> prep(const optional<Tensor> &t) {
  if (!t.has_value()) return t;
  return prep(*t);
}

kda_tensor desc(const Tensor *t) {
  kda_tensor d{nullptr, 0, 0, 0, 0};
  if (t == nullptr) return d;
  int64_t st[4];
  for (int i = 0; i < 4; ++i) st[i] = t->size(i) == 1 ? 0 : t->stride(i);
  d.data = t->data_ptr();
  d.stride_b = st[0];
  d.stride_h = st[1];
  d.stride_t = st[2];
  d.stride_d = 1;
  return d;
}

void *ptr(const Tensor *t) { return (t == nullptr || t->numel() == 0) ? nullptr : t->data_ptr(); }

int32_t dtype_code(const Tensor &q) {
  if (q.scalar_type() == at::kBFloat16) return KDA_DTYPE_BF16;
  if (q.scalar_type() == at::kHalf) return KDA_DTYPE_F16;
  TORCH_CHECK(false, "KDA sm_100a kernels take bf16/fp16 inputs, got ", q.scalar_type());
}

// per-device int32 word the kernels OR device-side error bits into (shared with Python)
std::mutex g_status_mu;
std::vector<Tensor> g_status;

Tensor status_word(const at::Device &dev) {
  std::lock_guard<std::mutex> lock(g_status_mu);
  const int idx = dev.index();
  if ((int)g_status.size() <= idx) g_status.resize(idx + 1);
  if (!g_status[idx].defined())
    g_status[idx] = at::zeros({1}, at::TensorOptions().dtype(at::kInt).device(at::kCUDA, idx));
  return g_status[idx];
}

void decay_fields(const optional<Tensor> &decay, const float **p, int64_t *sb, int64_t *sh, int64_t *sd) {
  *p = nullptr;
  *sb = *sh = *sd = 0;
  if (!decay.has_value()) return;
  const Tensor &d = *decay;
  TORCH_CHECK(d.dim() == 3 && d.scalar_type() == at::kFloat, "decay must be a float32 [B, H, D] view");
  *p = d.data_ptr<float>();
  *sb = d.size(0) == 1 ? 0 : d.stride(0);
  *sh = d.size(1) == 1 ? 0 : d.stride(1);
  *sd = d.size(2) == 1 ? 0 : d.stride(2);
}

// state-update semantics of the ops: 0 = K^T V (chunk-constant decay), 1 = the
// reference's literal K V^T, 2 = per-token decay
// Error messages format integers with std::to_string, never by streaming them
// into a std::ostream (which TORCH_CHECK does with its arguments): with this
// toolchain and torch build, an integer streamed inside an extension module
// crashed the process (SIGSEGV) instead of raising.
uint32_t mode_flags(int64_t mode) {
  TORCH_CHECK(mode >= 0 && mode <= 2, "mode must be 0 (corrected), 1 (literal) or 2 (per-step), got ",
              std::to_string(mode));
  return mode == 1 ? KDA_FLAG_LITERAL : (mode == 2 ? KDA_FLAG_PER_STEP : 0u);
}

void check(int rc, const char *what) {
  TORCH_CHECK(rc == KDA_OK, what, " failed: ", kda_status_string(rc), " (status ", std::to_string(rc), ")");
}

void check_inputs(const Tensor &q, const Tensor &k, const Tensor &v, const optional<Tensor> &g) {
  TORCH_CHECK(q.is_cuda(), "the KDA sm_100a kernels need CUDA tensors (there is no CPU path)");
  TORCH_CHECK(q.dim() == 4, "q must be [B, H, T, D]");
  auto same = [&](const Tensor &t, const char *n) {
    TORCH_CHECK(t.sizes() == q.sizes(), n, " shape must match q");
    TORCH_CHECK(t.scalar_type() == q.scalar_type() && t.device() == q.device(), n,
                " must match q's dtype and device");
  };
  same(k, "k");
  same(v, "v");
  if (g.has_value()) same(*g, "gate");
}

std::tuple<Tensor, Tensor> chunk_fwd(const Tensor &q_, const Tensor &k_, const Tensor &v_,
                                     const optional<Tensor> &g_, const optional<Tensor> &decay,
                                     double decay_scalar, const optional<Tensor> &s0, int64_t chunk, int64_t mode,
                                     bool want_state) {
  check_inputs(q_, k_, v_, g_);
  c10::cuda::CUDAGuard guard(q_.device());
  const Tensor q = prep(q_), k = prep(k_), v = prep(v_);
  const optional<Tensor> g = prep(g_);
  const int64_t B = q.size(0), H = q.size(1), T = q.size(2), D = q.size(3);
  const Tensor y = prep(empty_in_order_of(q));  // like the reference: keeps q's memory order
  const auto f32 = q.options().dtype(at::kFloat);
  const Tensor s_out = want_state ? at::empty({B, H, D, D}, f32) : at::empty({0}, f32);
  const optional<Tensor> s_in = s0.has_value() ? optional<Tensor>(s0->contiguous().to(at::kFloat)) : c10::nullopt;
  const uint32_t flags = mode_flags(mode);
  const size_t ws_bytes = kda_fwd_workspace_bytes((int32_t)B, (int32_t)H, (int32_t)T, (int32_t)D, (int32_t)chunk, flags);
  const Tensor ws = at::empty({(int64_t)ws_bytes}, q.options().dtype(at::kByte));
  kda_fwd_params p{};
  p.B = (int32_t)B; p.H = (int32_t)H; p.T = (int32_t)T; p.D = (int32_t)D; p.chunk = (int32_t)chunk;
  p.dtype = dtype_code(q);
  p.flags = flags;
  p.q = desc(&q); p.k = desc(&k); p.v = desc(&v); p.g = desc(g.has_value() ? &*g : nullptr); p.y = desc(&y);
  decay_fields(decay, &p.decay, &p.decay_stride_b, &p.decay_stride_h, &p.decay_stride_d);
  p.decay_scalar = decay_scalar;
  p.state_in = s_in.has_value() ? static_cast<const float *>(ptr(&*s_in)) : nullptr;
  p.state_out = want_state ? static_cast<float *>(ptr(&s_out)) : nullptr;
  p.workspace = ptr(&ws);
  p.workspace_bytes = ws_bytes;
  p.status = status_word(q.device()).data_ptr<int32_t>();
  check(kda_fwd_sm100(&p, c10::cuda::getCurrentCUDAStream(q.device().index()).stream()), "kda_fwd_sm100");
  return {y, s_out};
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> chunk_bwd(
    const Tensor &q_, const Tensor &k_, const Tensor &v_, const optional<Tensor> &g_, const Tensor &dy_,
    const optional<Tensor> &decay, double decay_scalar, const optional<Tensor> &s0, const optional<Tensor> &s_T,
    const optional<Tensor> &ds_T, int64_t chunk, int64_t mode, bool need_ddecay_, bool need_ds0) {
  (void)s_T;
  check_inputs(q_, k_, v_, g_);
  c10::cuda::CUDAGuard guard(q_.device());
  const Tensor q = prep(q_), k = prep(k_), v = prep(v_), dy = prep(dy_);
  const optional<Tensor> g = prep(g_);
  const int64_t B = q.size(0), H = q.size(1), T = q.size(2), D = q.size(3);
  const Tensor dq = prep(empty_in_order_of(q)), dk = prep(empty_in_order_of(k)), dv = prep(empty_in_order_of(v));
  const Tensor dg = g.has_value() ? prep(empty_in_order_of(*g)) : at::empty({0}, q.options());
  const bool need_ddecay = need_ddecay_ && decay.has_value();
  const auto f32 = q.options().dtype(at::kFloat);
  const Tensor ddecay = need_ddecay ? at::empty({B, H, D}, f32) : at::empty({0}, f32);
  const Tensor ds0 = need_ds0 ? at::empty({B, H, D, D}, f32) : at::empty({0}, f32);
  const optional<Tensor> s_in = s0.has_value() ? optional<Tensor>(s0->contiguous().to(at::kFloat)) : c10::nullopt;
  const optional<Tensor> dsT = (ds_T.has_value() && ds_T->numel() > 0)
                                   ? optional<Tensor>(ds_T->contiguous().to(at::kFloat))
                                   : c10::nullopt;
  const uint32_t flags = mode_flags(mode);
  const size_t ws_bytes = kda_bwd_workspace_bytes((int32_t)B, (int32_t)H, (int32_t)T, (int32_t)D, (int32_t)chunk, flags);
  const Tensor ws = at::empty({(int64_t)ws_bytes}, q.options().dtype(at::kByte));
  kda_bwd_params p{};
  p.B = (int32_t)B; p.H = (int32_t)H; p.T = (int32_t)T; p.D = (int32_t)D; p.chunk = (int32_t)chunk;
  p.dtype = dtype_code(q);
  p.flags = flags;
  p.q = desc(&q); p.k = desc(&k); p.v = desc(&v); p.g = desc(g.has_value() ? &*g : nullptr); p.dy = desc(&dy);
  p.dq = desc(&dq); p.dk = desc(&dk); p.dv = desc(&dv); p.dg = desc(g.has_value() ? &dg : nullptr);
  decay_fields(decay, &p.decay, &p.decay_stride_b, &p.decay_stride_h, &p.decay_stride_d);
  p.decay_scalar = decay_scalar;
  p.state_in = s_in.has_value() ? static_cast<const float *>(ptr(&*s_in)) : nullptr;
  p.dstate_out = dsT.has_value() ? static_cast<const float *>(ptr(&*dsT)) : nullptr;
  p.dstate_in = need_ds0 ? static_cast<float *>(ptr(&ds0)) : nullptr;
  p.ddecay = need_ddecay ? static_cast<float *>(ptr(&ddecay)) : nullptr;
  p.workspace = ptr(&ws);
  p.workspace_bytes = ws_bytes;
  p.status = status_word(q.device()).data_ptr<int32_t>();
  check(kda_bwd_sm100(&p, c10::cuda::getCurrentCUDAStream(q.device().index()).stream()), "kda_bwd_sm100");
  return {dq, dk, dv, dg, ddecay, ds0};
}

// ------------------------------------------------------ the gated delta rule
int32_t gate_code(const Tensor &t, const char *n) {
  if (t.scalar_type() == at::kFloat) return KDA_DTYPE_F32;
  if (t.scalar_type() == at::kBFloat16) return KDA_DTYPE_BF16;
  if (t.scalar_type() == at::kHalf) return KDA_DTYPE_F16;
  TORCH_CHECK(false, n, " must be float32, bfloat16 or float16");
}

// 32-bit sizes of the C ABI
int32_t small(int64_t n) {
  TORCH_CHECK(n >= 0 && n <= 0x7fffffff, "delta rule: a size of ", std::to_string(n), " is out of range");
  return (int32_t)n;
}

bool index64(const Tensor &t, const char *n, const at::Device &dev) {
  TORCH_CHECK(t.dim() == 1 && (t.scalar_type() == at::kInt || t.scalar_type() == at::kLong) && t.device() == dev, n,
              " must be a one-dimensional int32 or int64 tensor on q's device");
  return t.scalar_type() == at::kLong;
}

// Sizes, inputs and gates of a chunked call; `hold` keeps what the pointers need alive.
kda_delta_params delta_params(const Tensor &q_, const Tensor &k_, const Tensor &v_, const Tensor &g, const Tensor &beta,
                              double scale, const optional<Tensor> &s0, const optional<Tensor> &cu,
                              std::vector<Tensor> &hold) {
  TORCH_CHECK(q_.is_cuda(), "the KDA sm_100a kernels need CUDA tensors (there is no CPU path)");
  TORCH_CHECK(q_.dim() == 4 && v_.dim() == 4 && k_.sizes() == q_.sizes(), "q, k must be [B, Hk, T, D], v [B, H, T, D]");
  TORCH_CHECK(q_.size(0) == v_.size(0) && q_.size(2) == v_.size(2) && q_.size(3) == v_.size(3),
              "q and v must have the same batch, tokens and head dim");
  TORCH_CHECK(g.sizes() == v_.sizes().slice(0, 3) && beta.sizes() == g.sizes(), "g and beta must be [B, H, T]");
  for (const Tensor *t : {&k_, &v_, &g, &beta})
    TORCH_CHECK(t->device() == q_.device(), "all tensors must be on q's device");
  TORCH_CHECK(k_.scalar_type() == q_.scalar_type() && v_.scalar_type() == q_.scalar_type(), "k and v must have q's dtype");
  const Tensor q = prep(q_), k = prep(k_), v = prep(v_);
  kda_delta_params p{};
  p.B = small(v.size(0)); p.H = small(v.size(1)); p.Hk = small(q.size(1)); p.T = small(v.size(2)); p.D = small(v.size(3));
  p.dtype = dtype_code(q);
  p.g_dtype = gate_code(g, "g");
  p.beta_dtype = gate_code(beta, "beta");
  p.scale = (float)scale;
  p.q = desc(&q); p.k = desc(&k); p.v = desc(&v);
  p.g = ptr(&g);
  p.beta = ptr(&beta);
  p.g_stride_b = g.stride(0); p.g_stride_h = g.stride(1); p.g_stride_t = g.stride(2);
  p.beta_stride_b = beta.stride(0); p.beta_stride_h = beta.stride(1); p.beta_stride_t = beta.stride(2);
  int64_t seqs = p.B;
  if (cu.has_value()) {
    p.cu_int64 = index64(*cu, "cu_seqlens", q.device()) ? 1 : 0;
    TORCH_CHECK(cu->numel() >= 1 && p.B == 1, "cu_seqlens needs at least one offset and a batch of 1");
    const Tensor c = cu->contiguous();
    p.cu_seqlens = c.data_ptr();
    seqs = c.numel() - 1;
    p.nseq = small(seqs);
    hold.push_back(c);
  }
  if (s0.has_value()) {
    TORCH_CHECK(s0->scalar_type() == at::kFloat && s0->device() == q.device() &&
                    s0->sizes() == at::IntArrayRef({seqs, (int64_t)p.H, (int64_t)p.D, (int64_t)p.D}),
                "initial_state must be float32 [sequences, H, D, D] on q's device");
    Tensor s = s0->contiguous();
    if (reinterpret_cast<uintptr_t>(s.data_ptr()) % 16) s = s.clone();
    p.state_in = static_cast<const float *>(ptr(&s));
    hold.push_back(s);
  }
  for (const Tensor &t : {q, k, v, g, beta}) hold.push_back(t);
  p.status = status_word(q.device()).data_ptr<int32_t>();
  return p;
}

int64_t delta_seqs(const kda_delta_params &p) { return p.cu_seqlens != nullptr ? p.nseq : p.B; }

std::tuple<Tensor, Tensor> delta_fwd(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &g,
                                     const Tensor &beta, double scale, const optional<Tensor> &s0,
                                     const optional<Tensor> &cu, bool want_state) {
  c10::cuda::OptionalCUDAGuard guard;
  if (q.is_cuda()) guard.set_device(q.device());
  std::vector<Tensor> hold;
  kda_delta_params p = delta_params(q, k, v, g, beta, scale, s0, cu, hold);
  const Tensor o = prep(empty_in_order_of(v));
  const auto f32 = q.options().dtype(at::kFloat);
  const Tensor s_out = want_state ? at::empty({delta_seqs(p), p.H, p.D, p.D}, f32) : at::empty({0}, f32);
  p.o = desc(&o);
  p.state_out = static_cast<float *>(ptr(&s_out));
  p.workspace_bytes = kda_delta_fwd_workspace_bytes(&p);
  const Tensor ws = at::empty({(int64_t)p.workspace_bytes}, q.options().dtype(at::kByte));
  p.workspace = ptr(&ws);
  check(kda_delta_fwd_sm100(&p, c10::cuda::getCurrentCUDAStream(q.device().index()).stream()), "kda_delta_fwd_sm100");
  return {o, s_out};
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> delta_bwd(
    const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &g, const Tensor &beta, double scale,
    const optional<Tensor> &s0, const optional<Tensor> &cu, const Tensor &dout_, const optional<Tensor> &ds_T,
    bool need_ds0) {
  c10::cuda::OptionalCUDAGuard guard;
  if (q.is_cuda()) guard.set_device(q.device());
  std::vector<Tensor> hold;
  kda_delta_params p = delta_params(q, k, v, g, beta, scale, s0, cu, hold);
  TORCH_CHECK(dout_.sizes() == v.sizes() && dout_.device() == q.device(), "dout must have v's shape and device");
  const Tensor dout = prep(dout_.scalar_type() == q.scalar_type() ? dout_ : dout_.to(q.scalar_type()));
  const Tensor dq = prep(empty_in_order_of(q)), dk = prep(empty_in_order_of(k)), dv = prep(empty_in_order_of(v));
  const Tensor dg = at::empty(g.sizes(), g.options()), dbeta = at::empty(beta.sizes(), beta.options());
  const auto f32 = q.options().dtype(at::kFloat);
  const Tensor ds0 = need_ds0 ? at::empty({delta_seqs(p), p.H, p.D, p.D}, f32) : at::empty({0}, f32);
  optional<Tensor> dsT;
  if (ds_T.has_value() && ds_T->numel() > 0) {
    TORCH_CHECK(ds_T->sizes() == at::IntArrayRef({delta_seqs(p), (int64_t)p.H, (int64_t)p.D, (int64_t)p.D}) &&
                    ds_T->device() == q.device(), "the final state's gradient has the wrong shape or device");
    dsT = ds_T->contiguous().to(at::kFloat);
    if (reinterpret_cast<uintptr_t>(dsT->data_ptr()) % 16) dsT = dsT->clone();
    p.dstate_out = static_cast<const float *>(ptr(&*dsT));
  }
  p.dout = desc(&dout);
  p.dq = desc(&dq); p.dk = desc(&dk); p.dv = desc(&dv);
  p.dg = ptr(&dg);
  p.dbeta = ptr(&dbeta);
  p.dstate_in = static_cast<float *>(ptr(&ds0));
  p.workspace_bytes = kda_delta_bwd_workspace_bytes(&p);
  const Tensor ws = at::empty({(int64_t)p.workspace_bytes}, q.options().dtype(at::kByte));
  p.workspace = ptr(&ws);
  check(kda_delta_bwd_sm100(&p, c10::cuda::getCurrentCUDAStream(q.device().index()).stream()), "kda_delta_bwd_sm100");
  return {dq, dk, dv, dg, dbeta, ds0};
}

Tensor delta_step(const Tensor &q_, const Tensor &k_, const Tensor &v_, const Tensor &g, const Tensor &beta,
                  Tensor &state, const optional<Tensor> &slots, double scale) {
  TORCH_CHECK(q_.is_cuda(), "the KDA sm_100a kernels need CUDA tensors (there is no CPU path)");
  TORCH_CHECK(q_.dim() == 3 && v_.dim() == 3 && k_.sizes() == q_.sizes() && q_.size(0) == v_.size(0) &&
                  q_.size(2) == v_.size(2), "q, k must be [N, Hk, D], v [N, H, D]");
  TORCH_CHECK(g.sizes() == v_.sizes().slice(0, 2) && beta.sizes() == g.sizes(), "g and beta must be [N, H]");
  for (const Tensor *t : {&k_, &v_, &g, &beta, const_cast<const Tensor *>(&state)})
    TORCH_CHECK(t->device() == q_.device(), "all tensors must be on q's device");
  TORCH_CHECK(k_.scalar_type() == q_.scalar_type() && v_.scalar_type() == q_.scalar_type(), "k and v must have q's dtype");
  const int64_t N = v_.size(0), H = v_.size(1), D = v_.size(2);
  TORCH_CHECK(state.dim() == 4 && state.scalar_type() == at::kFloat && state.size(1) == H && state.size(2) == D &&
                  state.size(3) == D, "state must be float32 [states, H, D, D]");
  // a dimension of one element is never stepped over, whatever stride it reports
  auto st = [](const Tensor &t, int i) { return t.size(i) == 1 ? (int64_t)0 : t.stride(i); };
  // one of the two dimensions steps over all that the other spans
  const int64_t states = state.size(0), sn = st(state, 0), sh = st(state, 1);
  const bool apart = (states == 1 || sn >= D * D) && (H == 1 || sh >= D * D) &&
                     (states == 1 || H == 1 || sn >= (H - 1) * sh + D * D || sh >= (states - 1) * sn + D * D);
  TORCH_CHECK(state.numel() == 0 || (state.stride(3) == 1 && state.stride(2) == D && sn % 4 == 0 && sh % 4 == 0 && apart &&
                                     reinterpret_cast<uintptr_t>(state.data_ptr()) % 16 == 0),
              "state is updated in place: each [D, D] must be contiguous, 16-byte aligned and apart from the others");
  c10::cuda::CUDAGuard guard(q_.device());
  const Tensor q = prep(q_), k = prep(k_), v = prep(v_);
  Tensor o = at::empty({N, H, D}, v.options());
  kda_delta_step_params p{};
  p.N = small(N); p.H = small(H); p.Hk = small(q.size(1)); p.D = small(D); p.num_states = small(state.size(0));
  p.dtype = dtype_code(q);
  p.g_dtype = gate_code(g, "g");
  p.beta_dtype = gate_code(beta, "beta");
  p.scale = (float)scale;
  p.q = ptr(&q); p.k = ptr(&k); p.v = ptr(&v); p.o = ptr(&o); p.g = ptr(&g); p.beta = ptr(&beta);
  p.q_stride_n = st(q, 0); p.q_stride_h = st(q, 1);
  p.k_stride_n = st(k, 0); p.k_stride_h = st(k, 1);
  p.v_stride_n = st(v, 0); p.v_stride_h = st(v, 1);
  p.o_stride_n = st(o, 0); p.o_stride_h = st(o, 1);
  p.g_stride_n = g.stride(0); p.g_stride_h = g.stride(1);
  p.beta_stride_n = beta.stride(0); p.beta_stride_h = beta.stride(1);
  p.state = static_cast<float *>(ptr(&state));
  p.state_stride_n = sn;
  p.state_stride_h = sh;
  Tensor idx;
  if (slots.has_value()) {
    p.slots_int64 = index64(*slots, "state_indices", q.device()) ? 1 : 0;
    TORCH_CHECK(slots->size(0) == N, "state_indices must be [N]");
    idx = slots->contiguous();
    p.slots = ptr(&idx);
  } else {
    TORCH_CHECK(N <= state.size(0), "without state_indices there must be a state for each row");
  }
  p.status = status_word(q.device()).data_ptr<int32_t>();
  check(kda_delta_step_sm100(&p, c10::cuda::getCurrentCUDAStream(q.device().index()).stream()), "kda_delta_step_sm100");
  return o;
}

// The status word the kernels write (Python reads and clears it).
Tensor status(int64_t device) { return status_word(at::Device(at::kCUDA, (c10::DeviceIndex)device)); }

// ------------------------------------------------ fused elementwise / row ops
int32_t dtype16(const Tensor &t) {
  TORCH_CHECK(t.is_cuda(), "the sm_100a fused ops need CUDA tensors (there is no CPU path)");
  return dtype_code(t);
}
cudaStream_t stream_of(const Tensor &t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

Tensor silu_mul(const Tensor &a_, const Tensor &b_) {
  TORCH_CHECK(a_.sizes() == b_.sizes() && a_.scalar_type() == b_.scalar_type(), "silu_mul: a and b must match");
  c10::cuda::CUDAGuard guard(a_.device());
  const Tensor a = a_.contiguous(), b = b_.contiguous();
  Tensor out = at::empty_like(a);
  check(st_silu_mul_fwd(a.data_ptr(), b.data_ptr(), out.data_ptr(), a.numel(), dtype16(a), stream_of(a)),
        "st_silu_mul_fwd");
  return out;
}

std::tuple<Tensor, Tensor> silu_mul_bwd(const Tensor &a_, const Tensor &b_, const Tensor &g_) {
  c10::cuda::CUDAGuard guard(a_.device());
  const Tensor a = a_.contiguous(), b = b_.contiguous(), g = g_.contiguous().to(a.scalar_type());
  Tensor da = at::empty_like(a), db = at::empty_like(b);
  check(st_silu_mul_bwd(a.data_ptr(), b.data_ptr(), g.data_ptr(), da.data_ptr(), db.data_ptr(), a.numel(),
                        dtype16(a), stream_of(a)),
        "st_silu_mul_bwd");
  return {da, db};
}

std::tuple<Tensor, Tensor> rmsnorm_residual(const Tensor &x_, const Tensor &r_, const Tensor &w_, double eps) {
  TORCH_CHECK(x_.sizes() == r_.sizes(), "rmsnorm_residual: x and residual must match");
  TORCH_CHECK(w_.dim() == 1 && w_.size(0) == x_.size(-1), "rmsnorm_residual: weight must be [D]");
  c10::cuda::CUDAGuard guard(x_.device());
  const Tensor x = x_.contiguous(), r = r_.contiguous().to(x.scalar_type()), w = w_.contiguous().to(x.scalar_type());
  const int64_t D = x.size(-1), N = D ? x.numel() / D : 0;
  Tensor out = at::empty_like(x);
  Tensor rstd = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
  check(st_rmsnorm_residual_fwd(x.data_ptr(), r.data_ptr(), w.data_ptr(), out.data_ptr(), rstd.data_ptr<float>(), N,
                                D, (float)eps, dtype16(x), stream_of(x)),
        "st_rmsnorm_residual_fwd");
  return {out, rstd};
}

std::tuple<Tensor, Tensor> rmsnorm_residual_bwd(const Tensor &x_, const Tensor &w_, const Tensor &rstd_,
                                                const Tensor &dy_) {
  c10::cuda::CUDAGuard guard(x_.device());
  const Tensor x = x_.contiguous(), w = w_.contiguous().to(x.scalar_type()), rstd = rstd_.contiguous(),
               dy = dy_.contiguous().to(x.scalar_type());
  const int64_t D = x.size(-1), N = D ? x.numel() / D : 0;
  Tensor dx = at::empty_like(x);
  Tensor dw = at::empty({D}, x.options().dtype(at::kFloat));
  Tensor scratch = at::empty({(int64_t)(st_rmsnorm_residual_bwd_scratch(N, D) / sizeof(float)) + 1},
                             x.options().dtype(at::kFloat));
  check(st_rmsnorm_residual_bwd(x.data_ptr(), w.data_ptr(), rstd.data_ptr<float>(), dy.data_ptr(), dx.data_ptr(),
                                dw.data_ptr<float>(), scratch.data_ptr<float>(), N, D, dtype16(x), stream_of(x)),
        "st_rmsnorm_residual_bwd");
  return {dx, dw};
}

std::tuple<Tensor, Tensor, Tensor> cross_entropy(const Tensor &logits_, const Tensor &labels_, bool want_probs) {
  TORCH_CHECK(logits_.dim() == 2, "cross_entropy: logits must be [N, V]");
  TORCH_CHECK(labels_.dim() == 1 && labels_.size(0) == logits_.size(0), "cross_entropy: labels must be [N]");
  c10::cuda::CUDAGuard guard(logits_.device());
  const Tensor logits = logits_.contiguous(), labels = labels_.contiguous().to(at::kLong);
  const int64_t N = logits.size(0), V = logits.size(1);
  const auto f32 = logits.options().dtype(at::kFloat);
  Tensor loss = at::empty({N}, f32), lse = at::empty({N}, f32);
  Tensor probs = want_probs ? at::empty_like(logits) : at::empty({0}, logits.options());
  check(st_cross_entropy_fwd(logits.data_ptr(), labels.data_ptr<int64_t>(), loss.data_ptr<float>(),
                             lse.data_ptr<float>(), want_probs ? probs.data_ptr() : nullptr, N, V, dtype16(logits),
                             stream_of(logits)),
        "st_cross_entropy_fwd");
  return {loss, lse, probs};
}

Tensor cross_entropy_bwd(const Tensor &logits_, const Tensor &labels_, const Tensor &lse_, const Tensor &dloss_) {
  c10::cuda::CUDAGuard guard(logits_.device());
  const Tensor logits = logits_.contiguous(), labels = labels_.contiguous().to(at::kLong), lse = lse_.contiguous(),
               dloss = dloss_.contiguous().to(at::kFloat);
  const int64_t N = logits.size(0), V = logits.size(1);
  Tensor dlogits = at::empty_like(logits);
  check(st_cross_entropy_bwd(logits.data_ptr(), labels.data_ptr<int64_t>(), lse.data_ptr<float>(),
                             dloss.data_ptr<float>(), dlogits.data_ptr(), N, V, dtype16(logits), stream_of(logits)),
        "st_cross_entropy_bwd");
  return dlogits;
}

int32_t logit_code(const Tensor &t) {
  TORCH_CHECK(t.is_cuda(), "the sm_100a fused ops need CUDA tensors (there is no CPU path)");
  return t.scalar_type() == at::kFloat ? (int32_t)ST_DTYPE_F32 : dtype_code(t);
}

// rows of V contiguous elements, any distance apart
Tensor logit_rows(const Tensor &t) {
  return (t.size(1) == 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1)) ? t : t.contiguous();
}
int64_t row_stride(const Tensor &t) { return t.size(0) <= 1 ? t.size(1) : t.stride(0); }

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> token_logprobs(const Tensor &logits_, const Tensor &tokens_,
                                                                  int64_t top_k, double temperature,
                                                                  int64_t ignore_index) {
  TORCH_CHECK(logits_.dim() == 2, "token_logprobs: logits must be [N, V]");
  TORCH_CHECK(tokens_.dim() == 1 && tokens_.size(0) == logits_.size(0) && tokens_.device() == logits_.device() &&
                  (tokens_.scalar_type() == at::kLong || tokens_.scalar_type() == at::kInt),
              "token_logprobs: tokens must be int32 or int64 [N] on the logits' device");
  const int32_t dt = logit_code(logits_);
  const int64_t N = logits_.size(0), V = logits_.size(1);
  TORCH_CHECK(top_k >= 0 && top_k <= 32 && top_k <= V, "token_logprobs: top_k must be in [0, min(32, V)], got ",
              std::to_string(top_k));
  c10::cuda::CUDAGuard guard(logits_.device());
  const Tensor logits = logit_rows(logits_), tokens = tokens_.contiguous().to(at::kLong);
  const auto f32 = logits.options().dtype(at::kFloat);
  Tensor lp = at::empty({N}, f32), ent = at::empty({N}, f32), lse = at::empty({N}, logits.options().dtype(at::kDouble));
  Tensor top = at::empty({N, top_k}, f32), ids = at::empty({N, top_k}, tokens.options());
  check(st_token_logprobs_fwd(logits.data_ptr(), row_stride(logits), tokens.data_ptr<int64_t>(), lp.data_ptr<float>(),
                              ent.data_ptr<float>(), lse.data_ptr<double>(), static_cast<float *>(ptr(&top)),
                              static_cast<int64_t *>(ptr(&ids)), (int32_t)top_k, N, V, (float)temperature, ignore_index,
                              dt, stream_of(logits)),
        "st_token_logprobs_fwd");
  return {lp, ent, lse, top, ids};
}

Tensor token_logprobs_bwd(const Tensor &logits_, const Tensor &tokens_, const Tensor &ent_, const Tensor &lse_,
                          const optional<Tensor> &dlp_, const optional<Tensor> &dent_, double temperature,
                          int64_t ignore_index) {
  c10::cuda::CUDAGuard guard(logits_.device());
  const int64_t N = logits_.size(0), V = logits_.size(1);
  const Tensor logits = logit_rows(logits_), tokens = tokens_.contiguous().to(at::kLong), ent = ent_.contiguous(),
               lse = lse_.contiguous();
  auto upstream = [](const optional<Tensor> &t) { return t.has_value() ? t->contiguous().to(at::kFloat) : Tensor(); };
  const Tensor dlp = upstream(dlp_), dent = upstream(dent_);
  Tensor dlogits = at::empty({N, V}, logits.options());
  check(st_token_logprobs_bwd(logits.data_ptr(), row_stride(logits), tokens.data_ptr<int64_t>(), ent.data_ptr<float>(),
                              lse.data_ptr<double>(), dlp.defined() ? dlp.data_ptr<float>() : nullptr,
                              dent.defined() ? dent.data_ptr<float>() : nullptr, dlogits.data_ptr(), N, V,
                              (float)temperature, ignore_index, logit_code(logits), stream_of(logits)),
        "st_token_logprobs_bwd");
  return dlogits;
}

// ------------------------------------------------------------------ autograd
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

// Whether a call has to be recorded; without that it goes straight to the kernels (an autograd node
// costs a call 5 us of host time).  A forward-mode tangent counts whatever the gradient mode: the
// node refuses it, where the kernels would leave it out.
bool has_tangent(const Tensor &t) { return t._fw_grad(/*level=*/0).defined(); }
bool recorded(std::initializer_list<const Tensor *> ts) {
  const bool grad = at::GradMode::is_enabled();
  for (const Tensor *t : ts)
    if (t != nullptr && ((grad && t->requires_grad()) || has_tangent(*t))) return true;
  return false;
}

// Gradients that cannot be differentiated again: under create_graph they carry an error for whoever tries.
variable_list once(variable_list grads, const char *what) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list live;
  for (Tensor &g : grads)
    if (g.defined()) live.push_back(g.detach().set_requires_grad(true));
  const auto error = std::make_shared<torch::autograd::DelayedError>(
      std::string(what) + " can be differentiated once only", (int64_t)live.size());
  live = (*error)(std::move(live));
  size_t i = 0;
  for (Tensor &g : grads)
    if (g.defined()) g = live[i++];
  return grads;
}

optional<Tensor> if_defined(const Tensor &t) { return t.defined() ? optional<Tensor>(t) : c10::nullopt; }

const auto &delta_fwd_op() {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("kda_b200::delta_fwd", "")
                             .typed<std::tuple<Tensor, Tensor>(const Tensor &, const Tensor &, const Tensor &, const Tensor &,
                                                               const Tensor &, double, const optional<Tensor> &,
                                                               const optional<Tensor> &, bool)>();
  return op;
}

struct DeltaFunction : public torch::autograd::Function<DeltaFunction> {
  static variable_list forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &g,
                               const Tensor &beta, double scale, const optional<Tensor> &s0, const optional<Tensor> &cu,
                               bool want_state) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [o, s] = delta_fwd_op().call(q, k, v, g, beta, scale, s0, cu, want_state);
    ctx->save_for_backward({q, k, v, g, beta, s0.has_value() ? *s0 : Tensor(), cu.has_value() ? *cu : Tensor()});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["state"] = want_state;
    ctx->set_materialize_grads(false);
    return {o, s};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const variable_list t = ctx->get_saved_variables();
    const Tensor &v = t[2];
    const bool need_ds0 = t[5].defined() && ctx->needs_input_grad(5);  // edges of the tensor arguments: the sixth
    const Tensor dout = grads[0].defined() ? grads[0] : at::zeros_like(v);
    const bool state = ctx->saved_data["state"].toBool() && grads[1].defined();
    static auto op = c10::Dispatcher::singleton()
                         .findSchemaOrThrow("kda_b200::delta_bwd", "")
                         .typed<std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor>(
                             const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &, double,
                             const optional<Tensor> &, const optional<Tensor> &, const Tensor &, const optional<Tensor> &,
                             bool)>();
    at::AutoDispatchBelowADInplaceOrView below;
    auto [dq, dk, dv, dg, db, ds0] =
        op.call(t[0], t[1], v, t[3], t[4], ctx->saved_data["scale"].toDouble(), if_defined(t[5]), if_defined(t[6]), dout,
                state ? optional<Tensor>(grads[1]) : c10::nullopt, need_ds0);
    return once({dq, dk, dv, dg, db, Tensor(), need_ds0 ? ds0 : Tensor(), Tensor(), Tensor()}, "gated_delta_chunk");
  }
};

std::tuple<Tensor, Tensor> delta_fwd_autograd(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &g,
                                              const Tensor &beta, double scale, const optional<Tensor> &s0,
                                              const optional<Tensor> &cu, bool want_state) {
  if (!recorded({&q, &k, &v, &g, &beta, s0.has_value() ? &*s0 : nullptr})) {
    at::AutoDispatchBelowADInplaceOrView below;
    return delta_fwd_op().call(q, k, v, g, beta, scale, s0, cu, want_state);
  }
  const variable_list r = DeltaFunction::apply(q, k, v, g, beta, scale, s0, cu, want_state);
  return {r[0], r[1]};
}

Tensor delta_step_autograd(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &g, const Tensor &beta,
                           Tensor &state, const optional<Tensor> &slots, double scale) {
  TORCH_CHECK_NOT_IMPLEMENTED(!recorded({&q, &k, &v, &g, &beta, const_cast<const Tensor *>(&state)}),
                              "gated_delta_step has no gradient: call it under torch.no_grad(), or differentiate "
                              "gated_delta_chunk");
  state.unsafeGetTensorImpl()->bump_version();  // a graph that saved the pool must notice
  at::AutoDispatchBelowADInplaceOrView below;
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("kda_b200::delta_step", "")
                       .typed<Tensor(const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &, Tensor &,
                                     const optional<Tensor> &, double)>();
  return op.call(q, k, v, g, beta, state, slots, scale);
}

const auto &token_logprobs_op() {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("st_b200::token_logprobs", "")
                             .typed<std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>(const Tensor &, const Tensor &, int64_t,
                                                                                       double, int64_t)>();
  return op;
}

struct LogprobsFunction : public torch::autograd::Function<LogprobsFunction> {
  static variable_list forward(AutogradContext *ctx, const Tensor &logits, const Tensor &tokens, int64_t top_k,
                               double temperature, int64_t ignore_index) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [lp, ent, lse, top, ids] = token_logprobs_op().call(logits, tokens, top_k, temperature, ignore_index);
    ctx->save_for_backward({logits, tokens, ent, lse});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["ignore_index"] = ignore_index;
    ctx->mark_non_differentiable({lse, top, ids});
    ctx->set_materialize_grads(false);
    return {lp, ent, lse, top, ids};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const variable_list t = ctx->get_saved_variables();
    static auto op = c10::Dispatcher::singleton()
                         .findSchemaOrThrow("st_b200::token_logprobs_bwd", "")
                         .typed<Tensor(const Tensor &, const Tensor &, const Tensor &, const Tensor &,
                                       const optional<Tensor> &, const optional<Tensor> &, double, int64_t)>();
    at::AutoDispatchBelowADInplaceOrView below;
    return once({op.call(t[0], t[1], t[2], t[3], if_defined(grads[0]), if_defined(grads[1]),
                         ctx->saved_data["temperature"].toDouble(), ctx->saved_data["ignore_index"].toInt()),
                 Tensor(), Tensor(), Tensor(), Tensor()},
                "token_logprobs");
  }
};

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> token_logprobs_autograd(const Tensor &logits, const Tensor &tokens,
                                                                           int64_t top_k, double temperature,
                                                                           int64_t ignore_index) {
  if (!recorded({&logits})) {
    at::AutoDispatchBelowADInplaceOrView below;
    return token_logprobs_op().call(logits, tokens, top_k, temperature, ignore_index);
  }
  const variable_list r = LogprobsFunction::apply(logits, tokens, top_k, temperature, ignore_index);
  return {r[0], r[1], r[2], r[3], r[4]};
}

}  // namespace

TORCH_LIBRARY(st_b200, m) {
  m.def("silu_mul(Tensor a, Tensor b) -> Tensor");
  m.def("silu_mul_bwd(Tensor a, Tensor b, Tensor dout) -> (Tensor, Tensor)");
  m.def("rmsnorm_residual(Tensor x, Tensor residual, Tensor weight, float eps) -> (Tensor, Tensor)");
  m.def("rmsnorm_residual_bwd(Tensor x, Tensor weight, Tensor rstd, Tensor dy) -> (Tensor, Tensor)");
  m.def("cross_entropy(Tensor logits, Tensor labels, bool want_probs) -> (Tensor, Tensor, Tensor)");
  m.def("cross_entropy_bwd(Tensor logits, Tensor labels, Tensor lse, Tensor dloss) -> Tensor");
  m.def(
      "token_logprobs(Tensor logits, Tensor tokens, int top_k, float temperature, int ignore_index) "
      "-> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def(
      "token_logprobs_bwd(Tensor logits, Tensor tokens, Tensor entropy, Tensor lse, Tensor? dlogprob, Tensor? dentropy, "
      "float temperature, int ignore_index) -> Tensor");
}

TORCH_LIBRARY_IMPL(st_b200, CUDA, m) {
  m.impl("silu_mul", &silu_mul);
  m.impl("silu_mul_bwd", &silu_mul_bwd);
  m.impl("rmsnorm_residual", &rmsnorm_residual);
  m.impl("rmsnorm_residual_bwd", &rmsnorm_residual_bwd);
  m.impl("cross_entropy", &cross_entropy);
  m.impl("cross_entropy_bwd", &cross_entropy_bwd);
  m.impl("token_logprobs", &token_logprobs);
  m.impl("token_logprobs_bwd", &token_logprobs_bwd);
}

TORCH_LIBRARY(kda_b200, m) {
  m.def(
      "chunk_fwd(Tensor q, Tensor k, Tensor v, Tensor? g, Tensor? decay, float decay_scalar, Tensor? s0, "
      "int chunk, int mode, bool want_state) -> (Tensor, Tensor)");
  m.def(
      "chunk_bwd(Tensor q, Tensor k, Tensor v, Tensor? g, Tensor dy, Tensor? decay, float decay_scalar, "
      "Tensor? s0, Tensor? s_T, Tensor? ds_T, int chunk, int mode, bool need_ddecay, bool need_ds0) "
      "-> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("status_word(int device) -> Tensor");
  m.def(
      "delta_fwd(Tensor q, Tensor k, Tensor v, Tensor g, Tensor beta, float scale, Tensor? s0, Tensor? cu_seqlens, "
      "bool want_state) -> (Tensor, Tensor)");
  m.def(
      "delta_bwd(Tensor q, Tensor k, Tensor v, Tensor g, Tensor beta, float scale, Tensor? s0, Tensor? cu_seqlens, "
      "Tensor dout, Tensor? ds_T, bool need_ds0) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def(
      "delta_step(Tensor q, Tensor k, Tensor v, Tensor g, Tensor beta, Tensor(a!) state, Tensor? state_indices, "
      "float scale) -> Tensor");
}

TORCH_LIBRARY_IMPL(kda_b200, CUDA, m) {
  m.impl("chunk_fwd", &chunk_fwd);
  m.impl("chunk_bwd", &chunk_bwd);
  m.impl("delta_fwd", &delta_fwd);
  m.impl("delta_bwd", &delta_bwd);
  m.impl("delta_step", &delta_step);
}

TORCH_LIBRARY_IMPL(kda_b200, CompositeExplicitAutograd, m) { m.impl("status_word", &status); }

TORCH_LIBRARY_IMPL(kda_b200, Autograd, m) {
  m.impl("delta_fwd", &delta_fwd_autograd);
  m.impl("delta_step", &delta_step_autograd);
}
TORCH_LIBRARY_IMPL(st_b200, Autograd, m) { m.impl("token_logprobs", &token_logprobs_autograd); }
