"""``token_logprobs`` against float64 (``oracle/delta_oracle.py``), forward and gradient.

Tolerances.  fp32 results come from sums in fp32 over at most 2^17 terms spread over
256 threads x 8 lanes of a row, from ex2 (2 units in the last place) and from
logarithms of magnitude up to 2^5: absolute 2^5 * 2^-22 = 2^-17 on log
probabilities and entropies, whatever the vocabulary.  A gradient in the logits'
type is p (a relative error of 2^-17 through the exponent's 2^-18 ... 2^-17) times
factors of the same error: 2^-15 in the 2-norm, plus half a step of a 16-bit type.
Two absolute parts: at the token the gradient is a (1 - p), off by a p 2^-17 however
small 1 - p is (V = 1: p = 1 and the gradient is 0), together 2^-17 |a|; and fp16 steps
by 2^-24 below 2^-14, so each element may be off by 2^-25, together 2^-25 sqrt(N V).
"""
import pytest
import torch

from oracle.delta_oracle import logprobs

pytestmark = pytest.mark.gpu
DEV = "cuda"
ABS = 2.0 ** -17


@pytest.fixture(autouse=True)
def _needs_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def half_step(dtype):
    return 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2


def make(N, V, dtype, seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    x = (spread * torch.randn(N, V, generator=g)).to(dtype).to(DEV)
    return x, torch.randint(0, V, (N,), generator=g).to(DEV), torch.randn(N, generator=g).to(DEV), \
        torch.randn(N, generator=g).to(DEV)


def check(x, tok, a, b, temperature, top_k=0):
    from simpletrain_b200.fused_ops import token_logprobs
    leaf = x.detach().requires_grad_(True)
    r = token_logprobs(leaf, tok, temperature=temperature, top_k=top_k)
    (dx,) = torch.autograd.grad((r.logprob, r.entropy), leaf, (a, b))
    ref = x.double().requires_grad_(True)
    lp, H = logprobs(ref, tok.long(), temperature)
    (dr,) = torch.autograd.grad((lp, H), ref, (a.double(), b.double()))
    assert (r.logprob.double() - lp).abs().max() <= ABS * max(1.0, lp.abs().max().item() / 32)
    assert (r.entropy.double() - H).abs().max() <= ABS
    assert dx.dtype == x.dtype and dx.shape == x.shape
    err = (dx.double() - dr).norm().item()
    least = 2.0 ** -17 * a.norm().item() + (2.0 ** -25 * dx.numel() ** 0.5 if x.dtype == torch.float16 else 0.0)
    assert err <= (2.0 ** -15 + half_step(x.dtype)) * dr.norm().item() + least, err
    if top_k:
        ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top_k]
        assert torch.equal(r.top_ids, ids)
        top = torch.log_softmax(x.double() / temperature, -1).gather(1, ids)
        assert (r.top_logprobs.double() - top).abs().max() <= ABS * max(1.0, top.abs().max().item() / 32)
    return r, dx


@pytest.mark.parametrize("N,V,dtype,k,t", [
    (1, 1, torch.float32, 1, 1.0), (3, 7, torch.bfloat16, 7, 0.5), (5, 33, torch.float16, 32, 1.0),
    (2, 1000, torch.bfloat16, 5, 1.3), (37, 1001, torch.float32, 20, 0.7), (1, 32000, torch.bfloat16, 32, 1.0),
    (4, 50257, torch.float32, 20, 0.9), (700, 4099, torch.float16, 3, 1.0), (9, 131072, torch.bfloat16, 32, 1.0),
])
def test_values_gradients_and_alternatives(N, V, dtype, k, t):
    x, tok, a, b = make(N, V, dtype)
    check(x, tok, a, b, t, k)


def test_masked_logits_rows_and_padding():
    from simpletrain_b200.fused_ops import token_logprobs
    x, tok, a, b = make(6, 5000, torch.float32)
    x[0, 3:] = -torch.inf          # three tokens left
    tok[0] = 1
    x[1] = -torch.inf              # nothing left
    x[2] = 2.5                     # all equal: the lowest ids first
    x[3] = torch.finfo(torch.float32).min
    x[3, 17] = 0.0
    tok[3] = 17
    tok[4] = -100                  # padded
    tok[5] = 5000                  # names no token
    leaf = x.requires_grad_(True)
    r = token_logprobs(leaf, tok, top_k=5)
    (dx,) = torch.autograd.grad((r.logprob, r.entropy), leaf, (a, b))
    ref = x.detach()[0, :3].double()
    lp = torch.log_softmax(ref, -1)
    assert abs(r.logprob[0].item() - lp[1].item()) <= ABS
    assert abs(r.entropy[0].item() + (lp.exp() * lp).sum().item()) <= ABS
    order = torch.sort(ref, descending=True, stable=True).indices.tolist()
    assert r.top_ids[0].tolist() == order + [3, 4] and torch.isinf(r.top_logprobs[0, 3:]).all()
    assert torch.isfinite(dx[0]).all() and (dx[0, 3:] == 0).all()
    assert r.logprob[1].item() == -torch.inf and r.entropy[1].item() == 0 and (dx[1] == 0).all()
    assert r.top_ids[1].tolist() == [0, 1, 2, 3, 4]
    assert r.top_ids[2].tolist() == [0, 1, 2, 3, 4]
    assert abs(r.logprob[2].item() + torch.log(torch.tensor(5000.0)).item()) <= ABS
    assert r.logprob[3].item() == 0 and abs(r.entropy[3].item()) <= ABS and r.top_ids[3].tolist() == [17, 0, 1, 2, 3]
    assert r.logprob[4].item() == 0
    p = torch.softmax(x.detach()[4].double(), -1)
    want = -b[4].double() * p * (p.log() + r.entropy[4].double())
    assert (dx[4].double() - want).norm() <= 2.0 ** -15 * want.norm()
    assert torch.isnan(r.logprob[5]) and torch.isfinite(r.entropy[5])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masks_at_a_low_temperature(dtype):
    """A masked logit's gradient is 0 whatever 1 / temperature and the upstream gradient are."""
    x, tok, a, b = make(4, 3001, dtype, seed=5)
    x = (x.float() * 1e-4).to(dtype)
    x[:, 100:] = -torch.inf
    x[1, 100:] = torch.finfo(dtype).min
    check(x, tok % 100, a, 1e6 * b, 1e-4)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t,offset", [(1e-2, 0.0), (1e-3, 0.0), (1.0, 1e4), (1.0, -1e4), (1e-3, 300.0)])
def test_gradients_where_the_rows_sum_is_large(dtype, t, offset):
    """The probabilities keep their last bits when lse is large: logits over a low temperature, logits with a
    common offset.  A log probability's gradient sums to a (1 - sum p) / t over the row, at most 2^-15 |a| / t."""
    from simpletrain_b200.fused_ops import token_logprobs
    x, tok, a, b = make(6, 5003, dtype, seed=7)
    x = (x.float() + offset).to(dtype)
    tok[:3] = x[:3].argmax(-1)
    check(x, tok, a, b, t)
    leaf = x.float().requires_grad_(True)
    (dx,) = torch.autograd.grad(token_logprobs(leaf, tok, temperature=t).logprob, leaf, a)
    assert (dx.double().sum(-1).abs() <= 2.0 ** -15 * a.abs().double() / t).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("V", [3, 13, 33])
@pytest.mark.parametrize("t,offset", [(1e-2, 0.0), (1e-3, 100.0), (0.05, -1e4)])
def test_short_odd_rows_where_the_rows_sum_is_large(dtype, V, t, offset):
    """What lies before and behind a row's 16-byte vectors goes into the sums as exactly as the vectors do."""
    x, tok, a, b = make(64, V, dtype, seed=10, spread=max(3.0 * t, 1e-3))
    x = (x.float() + offset).to(dtype)
    ref = x.double()
    lp, H = logprobs(ref, tok, t)
    from simpletrain_b200.fused_ops import token_logprobs
    r = token_logprobs(x, tok, temperature=t, top_k=3)
    top = torch.log_softmax(ref / t, -1).gather(1, r.top_ids)
    assert (r.logprob.double() - lp).abs().max() <= ABS * max(1.0, lp.abs().max().item() / 32)
    assert (r.entropy.double() - H).abs().max() <= ABS
    assert (r.top_logprobs.double() - top).abs().max() <= ABS * max(1.0, top.abs().max().item() / 32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t", [0.5, 1.0, 2.0, 100.0])
def test_a_masked_logit_has_probability_0_at_every_temperature(dtype, t):
    from simpletrain_b200.fused_ops import token_logprobs
    x, tok, _, _ = make(3, 2500, dtype, seed=8)
    x[0, 2:] = torch.finfo(dtype).min
    x[1, 2:] = -2e29
    x[2, 2:] = -torch.inf
    tok[:] = 2
    r = token_logprobs(x, tok, temperature=t, top_k=4)
    assert (r.logprob == -torch.inf).all() and (r.top_logprobs[:, 2:] == -torch.inf).all()
    assert torch.isfinite(r.top_logprobs[:, :2]).all() and torch.isfinite(r.entropy).all()


def test_the_entropy_does_not_depend_on_the_token():
    """A token that names nothing makes its log probability NaN; the entropy alone and its gradient stay what they are."""
    from simpletrain_b200.fused_ops import token_logprobs
    x, tok, _, b = make(4, 1500, torch.float32, seed=9)
    bad = tok.clone()
    bad[1], bad[2] = -7, 1500
    got = []
    for t in (tok, bad):
        leaf = x.detach().requires_grad_(True)
        got.append(torch.autograd.grad(token_logprobs(leaf, t).entropy, leaf, b)[0])
    assert torch.equal(*got)
    leaf = x.detach().requires_grad_(True)
    (dx,) = torch.autograd.grad(token_logprobs(leaf, bad).logprob, leaf, b)
    assert torch.isnan(dx[1:3]).all() and torch.isfinite(dx[0]).all() and torch.isfinite(dx[3]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_lowest_values_as_masks(dtype):
    """A mask may be the type's lowest value; in fp16 that is a logit like others."""
    from simpletrain_b200.fused_ops import token_logprobs
    low = torch.finfo(dtype).min
    x, tok, a, b = make(4, 3001, dtype)
    x[0, 7:] = low
    x[1] = low
    x[2, ::2] = low
    x[2, 1::4] = -torch.inf
    x[3] = low
    x[3, 11] = -3.0
    tok = torch.tensor([3, 3, 3, 11], device=DEV)
    leaf = x.requires_grad_(True)
    r = token_logprobs(leaf, tok, top_k=2)
    (dx,) = torch.autograd.grad((r.logprob, r.entropy), leaf, (a, b))
    ref = x.detach().double()
    lp, H = logprobs(ref, tok)
    for n in (0, 2, 3):
        assert abs(r.logprob[n].item() - lp[n].item()) <= ABS and abs(r.entropy[n].item() - H[n].item()) <= ABS
    if dtype == torch.float16:
        assert abs(r.logprob[1].item() - lp[1].item()) <= ABS and abs(r.entropy[1].item() - H[1].item()) <= ABS
    else:
        assert r.logprob[1].item() == -torch.inf and r.entropy[1].item() == 0 and (dx[1] == 0).all()
    assert torch.isfinite(dx).all() and (dx[0, 7:] == 0).all() and (dx[2, ::2] == 0).all()
    assert r.top_ids[1].tolist() == [0, 1] and r.top_ids[3].tolist() == [11, 0]


def test_non_finite_logits_spoil_their_row_only():
    from simpletrain_b200.fused_ops import token_logprobs
    x, tok, _, _ = make(4, 20000, torch.bfloat16)
    clean = token_logprobs(x, tok, top_k=8)
    y = x.clone()
    y[1, 777] = torch.nan
    y[2, 19999] = torch.inf
    r = token_logprobs(y, tok, top_k=8)
    for n in (1, 2):
        assert torch.isnan(r.logprob[n]) and torch.isnan(r.entropy[n])
        assert ((r.top_ids[n] >= 0) & (r.top_ids[n] < 20000)).all()
    for n in (0, 3):
        for u, v in zip(clean, r):
            assert torch.equal(u[n], v[n])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_of_a_padded_vocabulary_and_odd_bases(dtype):
    g = torch.Generator().manual_seed(3)
    wide = (3 * torch.randn(5, 1040, generator=g)).to(dtype).to(DEV)
    flat = (3 * torch.randn(5 * 1003 + 1, generator=g)).to(dtype).to(DEV)
    tok = torch.randint(0, 1003, (5,), generator=g, dtype=torch.int32).to(DEV)
    a, b = torch.randn(5, generator=g).to(DEV), torch.randn(5, generator=g).to(DEV)
    for x in (wide[:, :1003], flat[1:].view(5, 1003), wide.t().contiguous().t()[:, :1003], wide[:, 5:6].expand(5, 1003)):
        check(x, tok, a, b, 1.0, 4)


def test_offsets_past_32_bits():
    from simpletrain_b200.fused_ops import token_logprobs
    N, V = 70000, 32003  # rows of odd length: every alignment
    gen = torch.Generator(device=DEV).manual_seed(4)
    x = torch.randn(N, V, generator=gen, device=DEV, dtype=torch.bfloat16)
    tok = torch.randint(0, V, (N,), generator=gen, device=DEV)
    up = torch.rand(N, generator=gen, device=DEV)
    got = []
    for pick in (slice(None), slice(N - 5, N)):
        leaf = x[pick].detach().requires_grad_(True)
        r = token_logprobs(leaf, tok[pick])
        (dx,) = torch.autograd.grad((r.logprob, r.entropy), leaf, (up[pick], up[pick]))
        got.append([t[-5:].clone() for t in (r.logprob, r.entropy, dx)])
        del r, dx
    # five rows are shared by more CTAs each: sums in another order
    assert (got[0][0] - got[1][0]).abs().max() <= ABS and (got[0][1] - got[1][1]).abs().max() <= ABS
    assert (got[0][2].double() - got[1][2].double()).norm() <= (2.0 ** -15 + 2 * half_step(x.dtype)) * got[1][2].double().norm()


def test_repeats_are_bitwise_equal_and_captured():
    from simpletrain_b200.fused_ops import token_logprobs
    x, tok, a, b = make(8, 32000, torch.bfloat16)
    leaf = x.requires_grad_(True)

    def step():
        r = token_logprobs(leaf, tok, top_k=10)
        return tuple(r) + torch.autograd.grad((r.logprob, r.entropy), leaf, (a, b))

    first = [t.detach().clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    graph.replay()
    torch.cuda.synchronize()
    for u, v in zip(first, out):
        assert torch.equal(u, v)


def test_empty_batch():
    from simpletrain_b200.fused_ops import token_logprobs
    x = torch.zeros(0, 100, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    r = token_logprobs(x, torch.zeros(0, device=DEV, dtype=torch.long), top_k=3)
    assert r.logprob.shape == (0,) and r.top_ids.shape == (0, 3)
    r.logprob.sum().backward()
    assert x.grad.shape == (0, 100)
