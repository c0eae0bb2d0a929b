"""The gated delta rule (``gated_delta_chunk``, ``gated_delta_step``) against its
definition in float64 (``oracle/delta_oracle.py``).

Tolerances, relative in the 2-norm.  Every operand of the kernels' products that is
not an input is carried in two 16-bit terms (a relative error of at most 2^-17 in
bf16, less in fp16) and every sum in fp32; a result goes through about four such
operands one after the other, so fp32 results are held to 4 * 2^-17 = 2^-15.  A
16-bit result is rounded once more, by at most eps/2 of each element.
"""
import pytest
import torch

from oracle.delta_oracle import gated_delta

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32_TOL = 2.0 ** -15
NAMES = ("q", "k", "v", "g", "beta")


@pytest.fixture(autouse=True)
def _needs_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def tol(dtype):
    return F32_TOL + (0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2)


def check(name, got, exp):
    assert got.shape == exp.shape, name
    got, ref = got.detach().double(), exp.detach().to(got.device)
    assert torch.isfinite(got).all(), name
    err, norm = (got - ref).norm().item(), ref.norm().item()
    assert err <= tol(exp_dtype(name, got, exp)) * norm + 1e-12, f"{name}: {err / max(norm, 1e-300):.3e}"


def exp_dtype(name, got, exp):
    return exp._lib_dtype


def as_result(ref, like):
    ref = ref.detach()
    ref._lib_dtype = like.dtype
    return ref


def make(B, H, Hk, T, D, dtype, gate, seed=0, decay=3.0, state=None, n=None):
    gen = torch.Generator().manual_seed(seed)

    def rnd(*s):
        return torch.randn(*s, generator=gen)

    def unit(*s):
        x = rnd(*s)
        return x / x.norm(dim=-1, keepdim=True)

    x = {"q": unit(B, T, Hk, D).to(dtype), "k": unit(B, T, Hk, D).to(dtype), "v": rnd(B, T, H, D).to(dtype),
         "g": torch.nn.functional.logsigmoid(rnd(B, T, H) + decay).to(gate), "beta": torch.sigmoid(rnd(B, T, H)).to(gate),
         "do": rnd(B, T, H, D).to(dtype)}
    x = {k_: t.to(DEV).transpose(1, 2) for k_, t in x.items()}
    n = B if n is None else n
    x["s0"] = (0.3 * rnd(n, H, D, D)).to(DEV) if state else None
    x["dsT"] = (0.3 * rnd(n, H, D, D)).to(DEV) if state else None
    return x


def run_both(x, D, cu=None, bounds=None, scale=None):
    """(library results, float64 results), each (o, final state, gradients...)."""
    from simpletrain_b200 import device_status, gated_delta_chunk
    outs = []
    for lib in (True, False):
        leaf = {n: x[n].detach().to(x[n].dtype if lib else torch.float64).requires_grad_(True) for n in NAMES}
        s0 = None if x["s0"] is None else x["s0"].detach().to(torch.float32 if lib else torch.float64).requires_grad_(True)
        if lib:
            o, s = gated_delta_chunk(*(leaf[n] for n in NAMES), initial_state=s0, cu_seqlens=cu, scale=scale)
        else:
            o, s = gated_delta(*(leaf[n] for n in NAMES), D ** -0.5 if scale is None else scale, s0, bounds)
        wrt = [leaf[n] for n in NAMES] + ([s0] if s0 is not None else [])
        ups = [x["do"].to(o.dtype)] + ([x["dsT"].to(s.dtype)] if s0 is not None else [])
        grads = torch.autograd.grad([o] + ([s] if s0 is not None else []), wrt, ups, allow_unused=True)
        outs.append([o, s] + [torch.zeros_like(w) if g is None else g for g, w in zip(grads, wrt)])
    torch.cuda.synchronize()
    assert device_status() == 0
    return outs


def compare(got, exp):
    for name, a, b in zip(("o", "state", "dq", "dk", "dv", "dg", "dbeta", "ds0"), got, exp):
        check(name, a, as_result(b, a))


CASES = [
    # B, H, Hk, T, D, dtype, gate dtype, state
    (1, 1, 1, 1, 64, torch.bfloat16, torch.float32, True),
    (1, 2, 2, 64, 64, torch.bfloat16, torch.float32, False),
    (2, 2, 1, 65, 64, torch.bfloat16, torch.bfloat16, True),
    (1, 2, 2, 63, 128, torch.bfloat16, torch.float32, True),
    (2, 3, 3, 130, 128, torch.bfloat16, torch.bfloat16, False),
    (1, 4, 2, 200, 128, torch.float16, torch.float16, True),
    (2, 6, 2, 257, 64, torch.float16, torch.float32, True),
    (1, 2, 1, 320, 128, torch.bfloat16, torch.float32, True),
]


@pytest.mark.parametrize("B,H,Hk,T,D,dtype,gate,state", CASES)
def test_forward_and_gradients(B, H, Hk, T, D, dtype, gate, state):
    x = make(B, H, Hk, T, D, dtype, gate, state=state)
    compare(*run_both(x, D))
