"""What the delta rule and the token log probabilities refuse, in Python and at the C ABI.
No kernel launches (runs without a GPU)."""
import ctypes

import pytest
import torch

from simpletrain_b200 import _ffi, gated_delta_chunk, gated_delta_step
from simpletrain_b200.fused_ops import token_logprobs


def chunk_args(B=2, H=4, Hk=2, T=5, D=64, dtype=torch.bfloat16, **change):
    a = dict(q=torch.zeros(B, Hk, T, D, dtype=dtype), k=torch.zeros(B, Hk, T, D, dtype=dtype),
             v=torch.zeros(B, H, T, D, dtype=dtype), g=torch.zeros(B, H, T), beta=torch.zeros(B, H, T))
    a.update(change)
    return a


@pytest.mark.parametrize("change,error", [
    (dict(), RuntimeError),                                             # CPU tensors
    (dict(q=torch.zeros(2, 2, 5, 64)), TypeError),                      # fp32 q
    (dict(k=torch.zeros(2, 2, 6, 64, dtype=torch.bfloat16)), ValueError),
    (dict(k=torch.zeros(2, 2, 5, 64, dtype=torch.float16)), TypeError),
    (dict(v=torch.zeros(2, 3, 5, 64, dtype=torch.bfloat16), g=torch.zeros(2, 3, 5), beta=torch.zeros(2, 3, 5)), ValueError),
    (dict(v=torch.zeros(2, 4, 5, 128, dtype=torch.bfloat16)), ValueError),
    (dict(g=torch.zeros(2, 4, 5, 1)), ValueError),
    (dict(beta=torch.zeros(2, 4)), ValueError),
    (dict(g=torch.zeros(2, 4, 5, dtype=torch.float64)), TypeError),
    (dict(initial_state=torch.zeros(2, 4, 64, 32)), ValueError),
    (dict(initial_state=torch.zeros(2, 4, 64, 64, dtype=torch.bfloat16)), TypeError),
    (dict(cu_seqlens=torch.tensor([0, 5])), ValueError),                # batch of 2
    (dict(cu_seqlens=torch.tensor([0.0, 5.0])), TypeError),
    (dict(cu_seqlens=torch.tensor([[0, 5]])), TypeError),
])
def test_chunk_refusals(change, error):
    with pytest.raises(error):
        gated_delta_chunk(**chunk_args(**change))


def test_chunk_refusals_of_packed_sequences():
    a = chunk_args(B=1)
    with pytest.raises(ValueError):
        gated_delta_chunk(**a, cu_seqlens=torch.zeros(0, dtype=torch.int32))
    long = {n: t[:, :, :1].expand(t.shape[0], t.shape[1], 2 ** 24 + 1, *t.shape[3:]) for n, t in a.items()}
    with pytest.raises(ValueError, match="2.24"):
        gated_delta_chunk(**long, cu_seqlens=torch.tensor([0, 5]))
    with pytest.raises(ValueError):  # three sequences, one state
        gated_delta_chunk(**a, cu_seqlens=torch.tensor([0, 1, 2, 5]), initial_state=torch.zeros(1, 4, 64, 64))


@pytest.mark.parametrize("D", [32, 96, 256])
def test_chunk_refuses_other_head_dims(D):
    with pytest.raises(ValueError):
        gated_delta_chunk(**chunk_args(D=D))


def step_args(N=3, H=4, Hk=2, D=64, S=5, **change):
    bf = torch.bfloat16
    a = dict(q=torch.zeros(N, Hk, D, dtype=bf), k=torch.zeros(N, Hk, D, dtype=bf), v=torch.zeros(N, H, D, dtype=bf),
             g=torch.zeros(N, H), beta=torch.zeros(N, H), state=torch.zeros(S, H, D, D))
    a.update(change)
    return a


@pytest.mark.parametrize("change,error", [
    (dict(), RuntimeError),
    (dict(state=torch.zeros(2, 4, 64, 64)), ValueError),                # fewer states than rows
    (dict(state=torch.zeros(5, 3, 64, 64)), ValueError),
    (dict(state=torch.zeros(5, 4, 64, 64, dtype=torch.float16)), TypeError),
    (dict(state_indices=torch.zeros(2, dtype=torch.int32)), ValueError),
    (dict(state_indices=torch.zeros(3)), TypeError),
    (dict(q=torch.zeros(3, 2, 1, 64, dtype=torch.bfloat16)), ValueError),
    (dict(g=torch.zeros(3, 2)), ValueError),
    (dict(state=torch.zeros(5, 4, 64, 64, requires_grad=True)), NotImplementedError),
])
def test_step_refusals(change, error):
    with pytest.raises(error):
        gated_delta_step(**step_args(**change))


@pytest.mark.parametrize("kw,error", [
    (dict(), RuntimeError),
    (dict(logits=torch.zeros(3)), ValueError),
    (dict(logits=torch.zeros(3, 0)), ValueError),
    (dict(logits=torch.zeros(3, 9, dtype=torch.float64)), TypeError),
    (dict(tokens=torch.zeros(2, dtype=torch.long)), ValueError),
    (dict(tokens=torch.zeros(3)), TypeError),
    (dict(top_k=10), ValueError),
    (dict(top_k=-1), ValueError),
    (dict(logits=torch.zeros(3, 99), top_k=33), ValueError),
    (dict(temperature=0.0), ValueError),
    (dict(temperature=float("nan")), ValueError),
])
def test_logprob_refusals(kw, error):
    a = dict(logits=torch.zeros(3, 9), tokens=torch.zeros(3, dtype=torch.long))
    a.update(kw)
    with pytest.raises(error):
        token_logprobs(a.pop("logits"), a.pop("tokens"), **a)


def test_forward_mode_derivatives_are_refused():
    """No tangent is computed, so none is left out silently (meta tensors: no kernel runs)."""
    import torch.autograd.forward_ad as fw
    bf = dict(dtype=torch.bfloat16, device="meta")

    def chunk(v):
        return gated_delta_chunk(torch.zeros(1, 2, 5, 64, **bf), torch.zeros(1, 2, 5, 64, **bf), v,
                                 torch.zeros(1, 2, 5, device="meta"), torch.zeros(1, 2, 5, device="meta"))[0]

    def step(v):
        return gated_delta_step(torch.zeros(3, 2, 64, **bf), torch.zeros(3, 2, 64, **bf), v, torch.zeros(3, 2, device="meta"),
                                torch.zeros(3, 2, device="meta"), torch.zeros(3, 2, 64, 64, device="meta"))

    def score(x):
        return token_logprobs(x, torch.zeros(3, dtype=torch.long, device="meta")).logprob

    for fn, x in ((chunk, torch.zeros(1, 2, 5, 64, **bf)), (step, torch.zeros(3, 2, 64, **bf)), (score, torch.zeros(3, 9, device="meta"))):
        assert fn(x).device.type == "meta"
        for mode in (torch.enable_grad, torch.no_grad):
            with mode(), fw.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
                fn(fw.make_dual(x, torch.ones_like(x)))
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.func.jvp(fn, (x,), (torch.ones_like(x),))


# ------------------------------------------------------------------ C ABI --
TENSOR = _ffi.KdaTensor(0x10000, 64 * 64, 64 * 64, 64, 1)


def delta_params(**kw):
    p = _ffi.KdaDeltaParams()
    p.B, p.H, p.Hk, p.T, p.D, p.scale = 1, 1, 1, 64, 64, 1.0
    p.q = p.k = p.v = p.o = p.dout = p.dq = p.dk = p.dv = TENSOR
    p.g = p.beta = p.dg = p.dbeta = 0x10000
    for n, v in kw.items():
        setattr(p, n, v)
    return p


@pytest.mark.parametrize("kw,code", [
    (dict(D=96), _ffi.KDA_ERR_UNSUPPORTED),
    (dict(dtype=2), _ffi.KDA_ERR_UNSUPPORTED),
    (dict(g_dtype=3), _ffi.KDA_ERR_UNSUPPORTED),
    (dict(H=3, Hk=2), _ffi.KDA_ERR_BAD_SHAPE),
    (dict(Hk=0), _ffi.KDA_ERR_BAD_SHAPE),
    (dict(T=-1), _ffi.KDA_ERR_BAD_SHAPE),
    (dict(H=70000, Hk=70000), _ffi.KDA_ERR_BAD_SHAPE),
    (dict(B=2, cu_seqlens=0x10000, nseq=1), _ffi.KDA_ERR_BAD_SHAPE),
    (dict(cu_seqlens=0x10000, nseq=-1), _ffi.KDA_ERR_BAD_SHAPE),
    (dict(T=2 ** 24 + 1, cu_seqlens=0x10000, nseq=1), _ffi.KDA_ERR_BAD_SHAPE),
    (dict(q=_ffi.KdaTensor(0x10008, 64, 64, 64, 1)), _ffi.KDA_ERR_BAD_LAYOUT),
    (dict(v=_ffi.KdaTensor(0x10000, 64, 64, 60, 1)), _ffi.KDA_ERR_BAD_LAYOUT),
    (dict(k=_ffi.KdaTensor(None, 64, 64, 64, 1)), _ffi.KDA_ERR_NULL_ARGUMENT),
    (dict(g=None), _ffi.KDA_ERR_NULL_ARGUMENT),
    (dict(state_in=0x10004), _ffi.KDA_ERR_BAD_LAYOUT),
    (dict(), _ffi.KDA_ERR_WORKSPACE),
    (dict(workspace=0x10080, workspace_bytes=1 << 30), _ffi.KDA_ERR_WORKSPACE),
    (dict(workspace=0x10000, workspace_bytes=100), _ffi.KDA_ERR_WORKSPACE),
    (dict(B=0), _ffi.KDA_OK),
    (dict(H=0, Hk=0), _ffi.KDA_OK),
])
def test_delta_abi_checks(kw, code):
    lib = _ffi.load()
    p = delta_params(**kw)
    assert lib.kda_delta_fwd_sm100(ctypes.byref(p), None) == code
    assert lib.kda_delta_bwd_sm100(ctypes.byref(p), None) == code
    assert lib.kda_delta_fwd_sm100(None, None) == _ffi.KDA_ERR_NULL_ARGUMENT


def test_delta_workspace_sizes():
    lib = _ffi.load()
    one = delta_params()
    f, b = lib.kda_delta_fwd_workspace_bytes(ctypes.byref(one)), lib.kda_delta_bwd_workspace_bytes(ctypes.byref(one))
    assert 0 < f < b
    # 64 tokens in n sequences are at most 1 + n chunks, each with 32 KB of T and P T
    few, many = (lib.kda_delta_fwd_workspace_bytes(ctypes.byref(delta_params(cu_seqlens=0x10000, nseq=n))) for n in (7, 15))
    assert few >= 8 * 32768 and many - few >= 8 * 32768
    assert lib.kda_delta_fwd_workspace_bytes(ctypes.byref(delta_params(D=96))) == 0


def test_workspace_of_padded_offsets():
    """Sequences beyond the tokens are empty: they need an offset each, no chunks."""
    lib = _ffi.load()
    for size in (lib.kda_delta_fwd_workspace_bytes, lib.kda_delta_bwd_workspace_bytes):
        few, many = (size(ctypes.byref(delta_params(H=8, Hk=8, cu_seqlens=0x10000, nseq=n))) for n in (64, 50000))
        assert 0 < few < many <= few + 2 * 4 * 50000 + 148 * 2 * 64 * 64 * 4 + 65536
    p = delta_params(H=8, Hk=8, cu_seqlens=0x10000, nseq=100000000)
    assert lib.kda_delta_fwd_workspace_bytes(ctypes.byref(p)) > 0


def step_params(**kw):
    p = _ffi.KdaDeltaStepParams()
    p.N, p.H, p.Hk, p.D, p.num_states, p.scale = 2, 2, 1, 64, 4, 1.0
    p.q = p.k = p.v = p.o = p.g = p.beta = p.state = 0x10000
    for n, v in kw.items():
        setattr(p, n, v)
    return p


@pytest.mark.parametrize("kw,code", [
    (dict(D=32), _ffi.KDA_ERR_UNSUPPORTED),
    (dict(dtype=2), _ffi.KDA_ERR_UNSUPPORTED),
    (dict(beta_dtype=-1), _ffi.KDA_ERR_UNSUPPORTED),
    (dict(H=3, Hk=2), _ffi.KDA_ERR_BAD_SHAPE),
    (dict(N=-1), _ffi.KDA_ERR_BAD_SHAPE),
    (dict(num_states=1), _ffi.KDA_ERR_BAD_SHAPE),
    (dict(q=None), _ffi.KDA_ERR_NULL_ARGUMENT),
    (dict(state=None), _ffi.KDA_ERR_NULL_ARGUMENT),
    (dict(v=0x10008), _ffi.KDA_ERR_BAD_LAYOUT),
    (dict(k_stride_n=4), _ffi.KDA_ERR_BAD_LAYOUT),
    (dict(state_stride_h=2), _ffi.KDA_ERR_BAD_LAYOUT),
    (dict(N=0), _ffi.KDA_OK),
])
def test_step_abi_checks(kw, code):
    assert _ffi.load().kda_delta_step_sm100(ctypes.byref(step_params(**kw)), None) == code


def test_logprob_abi_checks():
    lib = _ffi.load()
    P, I64, I32, F = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32, ctypes.c_float

    def fwd(logits=0x10000, stride=9, top=0x10000, k=1, N=2, V=9, t=1.0, dt=0):
        return lib.st_token_logprobs_fwd(P(logits), I64(stride), P(0x10000), P(0x10000), P(0x10000), P(0x10000), P(top), P(top),
                                         I32(k), I64(N), I64(V), F(t), I64(-100), I32(dt), P(None))

    assert fwd(k=33, V=99, stride=99) == _ffi.KDA_ERR_UNSUPPORTED
    assert fwd(k=10) == _ffi.KDA_ERR_BAD_SHAPE
    assert fwd(V=0) == _ffi.KDA_ERR_BAD_SHAPE
    assert fwd(stride=8) == _ffi.KDA_ERR_BAD_SHAPE
    assert fwd(t=0.0) == _ffi.KDA_ERR_UNSUPPORTED
    assert fwd(dt=3) == _ffi.KDA_ERR_UNSUPPORTED
    assert fwd(logits=None) == _ffi.KDA_ERR_NULL_ARGUMENT
    assert fwd(top=None) == _ffi.KDA_ERR_NULL_ARGUMENT
    assert fwd(logits=0x10001) == _ffi.KDA_ERR_BAD_LAYOUT
    assert fwd(N=0) == _ffi.KDA_OK
