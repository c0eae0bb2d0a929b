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
    # more streams than SMs: work ranges that cut streams, their states handed from CTA to CTA
    (5, 40, 20, 190, 64, torch.bfloat16, torch.float32, True),
    (10, 18, 18, 300, 128, torch.bfloat16, torch.bfloat16, True),
]


@pytest.mark.parametrize("B,H,Hk,T,D,dtype,gate,state", CASES)
def test_forward_and_gradients(B, H, Hk, T, D, dtype, gate, state):
    x = make(B, H, Hk, T, D, dtype, gate, state=state)
    compare(*run_both(x, D))


def packed(lens, lead=0, tail=0, dtype=torch.int32):
    ends = [lead]
    for n in lens:
        ends.append(ends[-1] + n)
    return torch.tensor(ends, dtype=dtype, device=DEV), list(zip(ends[:-1], ends[1:])), ends[-1] + tail


@pytest.mark.parametrize("lens,lead,tail,H,Hk,D,dtype,index", [
    ([70, 1, 0, 64, 129], 0, 0, 2, 2, 64, torch.bfloat16, torch.int32),
    ([0, 3, 200], 5, 9, 4, 2, 128, torch.bfloat16, torch.int64),
    ([1] * 40 + [0] * 3, 0, 70, 2, 1, 64, torch.float16, torch.int32),
    ([0], 0, 17, 1, 1, 128, torch.bfloat16, torch.int32),
    ([128], 0, 0, 2, 1, 128, torch.float16, torch.int32),
    ([7] * 50 + [900, 0, 64, 130] + [65] * 20, 3, 0, 4, 2, 64, torch.bfloat16, torch.int32),  # one stream over several ranges
])
def test_packed_sequences(lens, lead, tail, H, Hk, D, dtype, index):
    cu, bounds, T = packed(lens, lead, tail, index)
    x = make(1, H, Hk, T, D, dtype, torch.float32, seed=1, state=True, n=len(lens))
    with torch.no_grad():  # what lies outside the sequences is never used
        for n in ("q", "k", "v", "do"):
            x[n][:, :, :lead] = torch.nan
            x[n][:, :, T - tail:T] = torch.nan
            x[n][:, :, T - tail:T] = torch.inf if n == "v" else torch.nan
        for n in ("g", "beta"):
            x[n][:, :, :lead] = torch.nan
            x[n][:, :, T - tail:T] = torch.nan
    got, exp = run_both(x, D, cu, bounds)
    out = torch.ones(T, dtype=torch.bool, device=DEV)
    for lo, hi in bounds:
        out[lo:hi] = False
    for t in (got[0], *got[2:7]):
        assert (t[:, :, out] == 0).all()
    compare(got, exp)


@pytest.mark.parametrize("lens,H,Hk,D,dtype", [
    ([128] + [0] * 31, 8, 8, 64, torch.bfloat16),  # offsets padded with empty sequences, as a captured graph has them
    ([0] * 15 + [200], 10, 5, 128, torch.float16),
    ([0] * 9 + [129, 0, 0, 70] + [0] * 30, 6, 3, 64, torch.bfloat16),
    ([1, 0, 0, 2, 0] * 3 + [0] * 185, 2, 1, 64, torch.bfloat16),  # more sequences than tokens
])
def test_packed_with_fewer_chunks_than_ranges(lens, H, Hk, D, dtype):
    cu, bounds, T = packed(lens)
    x = make(1, H, Hk, T, D, dtype, torch.float32, seed=13, state=True, n=len(lens))
    compare(*run_both(x, D, cu, bounds))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_packed_row_without_tokens(dtype):
    from simpletrain_b200 import gated_delta_chunk
    x = make(1, 2, 2, 0, 64, dtype, torch.float32, state=True, n=5)
    leaf = [x[n].detach().requires_grad_(True) for n in (*NAMES, "s0")]
    o, s = gated_delta_chunk(*leaf[:5], initial_state=leaf[5], cu_seqlens=torch.zeros(6, dtype=torch.int32, device=DEV))
    assert o.shape == (1, 2, 0, 64) and torch.equal(s, x["s0"])
    assert torch.equal(torch.autograd.grad(s, leaf[5], x["dsT"])[0], x["dsT"])


def test_packed_rows_equal_their_own_calls():
    """A sequence's results do not depend on what it is packed with."""
    from simpletrain_b200 import gated_delta_chunk
    cu, bounds, T = packed([100, 64, 37])
    x = make(1, 2, 2, T, 128, torch.bfloat16, torch.float32, seed=2)
    x["v"][:, :, 100:164] = torch.nan  # a broken sequence between two others
    o, s = gated_delta_chunk(*(x[n] for n in NAMES), cu_seqlens=cu)
    for i, (lo, hi) in enumerate(bounds):
        oi, si = gated_delta_chunk(*(x[n][:, :, lo:hi] for n in NAMES))
        if i != 1:
            assert torch.equal(o[:, :, lo:hi], oi) and torch.equal(s[i], si[0])
    assert torch.isnan(o[:, :, 100:164]).any()


def test_fp16_results_do_not_depend_on_where_streams_are_cut():
    """A stream alone is one work range; among 200 others it is cut between CTAs.  The units that fp16 goes by are the same."""
    from simpletrain_b200 import gated_delta_chunk
    x = sized(make(3, 67, 67, 330, 64, torch.float16, torch.float32, seed=19, state=True), do=1e-3, v=3.0)
    results = []
    for pick in (slice(None), slice(1, 2)):
        leaf = [x[n][pick].detach().requires_grad_(True) for n in (*NAMES, "s0")]
        o, s = gated_delta_chunk(*leaf[:5], initial_state=leaf[5])
        results.append((o, s, *torch.autograd.grad([o, s], leaf, [x["do"][pick], x["dsT"][pick]])))
    for a, b in zip(*results):
        assert torch.equal(a[1:2], b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_zeros(dtype):
    """Nothing in, nothing out: no unit of zeros makes a NaN."""
    for zero in (("v", "s0"), ("do", "dsT"), ("q",), ("k",), ("beta",), ("v", "s0", "do", "dsT"), NAMES):
        x = make(1, 2, 1, 140, 64, dtype, torch.float32, seed=20, state=True)
        x = {n: torch.zeros_like(t) if n in zero else t for n, t in x.items()}
        compare(*run_both(x, 64))
    x = make(1, 2, 1, 140, 64, dtype, torch.float32, seed=20, state=True)
    compare(*run_both(x, 64, scale=0.0))


@pytest.mark.parametrize("value", [torch.nan, torch.inf])
def test_what_is_not_finite_stays_in_its_chunk_and_behind_in_fp16(value):
    from simpletrain_b200 import gated_delta_chunk
    for name in ("q", "k", "v"):
        x = make(1, 1, 1, 260, 64, torch.float16, torch.float32, seed=21)
        clean, s_clean = gated_delta_chunk(*(x[n] for n in NAMES))
        x[name][0, 0, 130, 3] = value
        leaf = [x[n].detach().requires_grad_(True) for n in NAMES]
        o, s = gated_delta_chunk(*leaf)
        assert torch.equal(o[:, :, :128], clean[:, :, :128]) and not torch.isfinite(o[0, 0, 130]).all()
        if name == "q":
            assert torch.equal(s, s_clean)
        else:
            assert not torch.isfinite(s).all()
        grads = torch.autograd.grad(o, leaf, x["do"])
        assert any(not torch.isfinite(g).all() for g in grads)


@pytest.mark.parametrize("name", NAMES)
def test_nan_is_not_swallowed(name):
    """A NaN of any input reaches the outputs from its token on, the state and the gradients."""
    from simpletrain_b200 import gated_delta_chunk
    x = make(1, 1, 1, 200, 64, torch.bfloat16, torch.float32)
    x[name][0, 0, 70] = torch.nan
    leaf = [x[n].detach().requires_grad_(True) for n in NAMES]
    o, s = gated_delta_chunk(*leaf)
    assert torch.isfinite(o[:, :, :64]).all() and torch.isnan(o[0, 0, 70]).all()
    if name != "q":
        assert torch.isnan(o[0, 0, 71:]).any(-1).all() and torch.isnan(s).any()
    grads = torch.autograd.grad(o, leaf, x["do"])
    assert any(torch.isnan(g).any() for g in grads)


@pytest.mark.parametrize("raw", [[0, 90, 40, 130], [-5, 20, 130, 131], [0, 10 ** 12, 60, 130], [200, 300, 400, 500]])
def test_bad_offsets_are_clamped_and_reported(raw):
    from simpletrain_b200 import _ffi, device_status, gated_delta_chunk
    T = 130
    x = make(1, 2, 2, T, 64, torch.bfloat16, torch.float32)
    clamped, most = [], 0
    for r in raw:
        most = max(most, min(max(r, 0), T))
        clamped.append(most)
    leaf = [x[n].requires_grad_(True) for n in NAMES]
    results = []
    for offsets in (raw, clamped):
        o, s = gated_delta_chunk(*leaf, cu_seqlens=torch.tensor(offsets, device=DEV))
        results.append((o, s, *torch.autograd.grad(o, leaf, x["do"])))
        assert device_status() == (_ffi.KDA_ERR_DEVICE_INDEX if offsets is raw else 0)
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("case", ["plain", "fused", "sliced", "broadcast", "misaligned"])
def test_layouts(case):
    """Results do not depend on strides; broadcast inputs get the sum of their gradients."""
    from simpletrain_b200 import gated_delta_chunk
    B, H, T, D = 2, 2, 75, 64
    x = make(B, H, H, T, D, torch.bfloat16, torch.float32, seed=3)
    base = {n: x[n].contiguous() for n in (*NAMES, "do")}
    if case == "broadcast":
        base["k"] = base["k"][:, :1].expand(B, H, T, D).contiguous()
        base["beta"] = base["beta"][:1].expand(B, H, T).contiguous()
    want = {n: base[n].clone().requires_grad_(True) for n in NAMES}
    o, s = gated_delta_chunk(*want.values())
    dw = torch.autograd.grad(o, list(want.values()), base["do"])
    if case == "plain":
        got = {n: base[n].clone().transpose(1, 2).contiguous().transpose(1, 2) for n in NAMES}
    elif case == "fused":
        proj = torch.stack([base[n].transpose(1, 2) for n in "qkv"], 2)  # [B, T, 3, H, D]
        got = dict(zip("qkv", (t.transpose(1, 2) for t in proj.unbind(2))), g=base["g"], beta=base["beta"])
    elif case == "sliced":
        got = {n: torch.cat([torch.full_like(base[n][:, :, :3], 9.0), base[n]], 2)[:, :, 3:] for n in NAMES}
    elif case == "broadcast":
        got = dict(base, k=base["k"][:, :1].expand(B, H, T, D), beta=base["beta"][:1].expand(B, H, T))
    else:
        got = {n: torch.cat([base[n].flatten()[:1], base[n].flatten()])[1:].view_as(base[n]) for n in NAMES}
    leaf = {n: got[n].detach().requires_grad_(True) for n in NAMES}
    o2, s2 = gated_delta_chunk(*(leaf[n] for n in NAMES))
    assert torch.equal(o, o2) and torch.equal(s, s2)
    dg = torch.autograd.grad(o2, [leaf[n] for n in NAMES], base["do"].transpose(2, 3).contiguous().transpose(2, 3))
    for n, a, b in zip(NAMES, dw, dg):
        assert torch.equal(a, b), n


def test_strong_and_absent_decay():
    """Resets (g far below 0, -inf), no decay at all, beta 0, 1 and 2."""
    x = make(1, 2, 2, 150, 64, torch.bfloat16, torch.float32, seed=4, state=True)
    x["g"][:, 0] = 0.0
    x["g"][:, 1, 40] = -1e4
    x["g"][:, 1, 90:93] = -torch.inf
    x["g"][:, 1, 127] = -60.0
    x["beta"][:, 0, 10:20] = 0.0
    x["beta"][:, 0, 30:60] = 1.0
    x["beta"][:, 0, 70:80] = 2.0
    got, exp = run_both(x, 64)
    # the gradient of a decay that is 0 in fp32 is 0; the formula's e^g at -inf and -1e4 is 0 too
    compare(got, exp)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("case", ["every other", "runs", "every third"])
def test_many_resets_in_a_chunk(case, D):
    """The running sum of the decay gets long; the factors between tokens after the resets keep their last bits."""
    x = make(1, 4, 2, 250, D, torch.float16, torch.float32, seed=3, state=True)
    if case == "every other":
        x["g"][..., ::2] = -110.0
    elif case == "runs":
        for i in range(4):
            x["g"][..., 64 * i:64 * i + 40] = -110.0
    else:
        x["g"][..., ::3] = -60.0
    compare(*run_both(x, D))


def sized(x, **by):
    """Inputs of `make` times a power of ten each, in their own types."""
    return {n: (t.double() * by[n]).to(t.dtype) if n in by and t is not None else t for n, t in x.items()}


def compare_sized(got, exp):
    """As compare(); fp16 steps by 2^-24 below 2^-14, so each element of a small result is off by up to 2^-25 more."""
    for name, a, b in zip(("o", "state", "dq", "dk", "dv", "dg", "dbeta", "ds0"), got, exp):
        dtype_of = a.dtype
        a, b = a.detach().double(), b.detach()
        if half := dtype_of == torch.float16:  # from 65520 on the nearest value of the type is infinity
            far = b.abs() >= 65520 * (1 + F32_TOL)
            assert (a[far] == b[far].sign() * torch.inf).all(), name
            fine = b.abs() <= 65520 * (1 - F32_TOL)
            a, b = a[fine], b[fine]
        assert torch.isfinite(a).all(), name
        err, norm = (a - b).norm().item(), b.norm().item()
        least = 2.0 ** -25 * a.numel() ** 0.5 if half else 0.0
        assert err <= tol(dtype_of) * norm + least, f"{name}: {err / max(norm, 1e-300):.3e}"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("by", [
    dict(do=1e-2, dsT=1e-2), dict(do=1e-4, dsT=1e-4), dict(do=1e-5, dsT=1e-5),  # a loss's mean without a loss scale
    dict(do=1e-5, dsT=1.0), dict(do=0.0, dsT=1e-8), dict(do=1e3, dsT=1e5, q=0.01),
    dict(v=1e-4, s0=1e-4), dict(v=1e-3, s0=1e-7), dict(s0=1e5, do=1e-3, dsT=1e-3), dict(v=300.0, do=1e-5, dsT=1e-5),
    dict(q=1e-2), dict(q=30.0, do=1e-2), dict(k=0.1), dict(k=0.1, beta=50.0), dict(k=1.4, do=1e-3, dsT=1e-3),
], ids=lambda by: " ".join(f"{n}={x:g}" for n, x in by.items()))
def test_sizes_of_the_inputs(by, dtype):
    """What the products' operands are rounded to does not depend on how large the inputs and the gradients are.
    fp16 carries them in units of a power of two a chunk, so that its range does not bound states and gradients."""
    x = sized(make(1, 2, 1, 300, 128, dtype, torch.float32, seed=14, state=True), **by)
    compare_sized(*run_both(x, 128))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_sizes_that_change_along_a_sequence(dtype):
    """Values of very different size in different chunks and sequences."""
    lens = [200, 64, 130, 70]
    cu, bounds, T = packed(lens)
    x = make(1, 4, 2, T, 64, dtype, torch.float32, seed=15, state=True, n=len(lens))
    x["v"][:, :, :64] *= 1e-3
    x["v"][:, :, 128:150] *= 1e3
    x["do"][:, :, :128] *= 1e-4
    x["g"][:, 1, 160] = -200.0
    x["s0"][1] *= 1e6
    x["s0"][2] = 0
    x["v"][:, :, 264:394] *= 1e-4
    x["do"][:, :, 264:394] *= 1e-4
    x["dsT"][3] *= 1e-6
    x["q"][:, :, 200:264] *= 1e-2
    got, exp = run_both(x, 64, cu, bounds)
    for i, (lo, hi) in enumerate(bounds):  # each sequence by itself: a large one does not hide a small one
        part = lambda r: [r[0][:, :, lo:hi], r[1][i], *(t[:, :, lo:hi] for t in r[2:7]), r[7][i]]
        compare_sized(part(got), part(exp))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("g", [-8.0, -20.0, -30.0])
def test_gradients_behind_strong_decays(g, dtype):
    """What a strong decay leaves of a state's gradient keeps its bits, however little it is.  (A chunk's first
    token has the strong gate, all of them, or the second chunk's first.)"""
    for pick in (slice(0, 1), slice(None), slice(64, 65)):
        x = make(1, 2, 1, 150, 64, dtype, torch.float32, seed=25, state=True)
        x["g"][:, :, pick] = g
        compare_sized(*run_both(x, 64))


def test_a_scale_far_from_the_default():
    for scale in (1e-4, 50.0):
        x = make(1, 2, 2, 150, 64, torch.float16, torch.float32, seed=16, state=True)
        x = sized(x, do=1e-2 / scale if scale > 1 else 1.0)
        compare_sized(*run_both(x, 64, scale=scale))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("beta", [1.0, 1.9])
@pytest.mark.parametrize("case", ["one key", "two keys", "near"])
def test_repeated_and_correlated_keys(case, beta, dtype):
    """(I + A)^-1 is largest where keys repeat.  For one key and no decay its rows are 1, -beta, -beta (1 - beta),
    -beta (1 - beta)^2 ...: an operand's error comes out of U = T X up to 1 + beta / (1 - |1 - beta|) times as large,
    2 for beta 1 and 20 for 1.9, and the fp32 part of the tolerance is that many times the others'."""
    x = make(1, 2, 1, 200, 64, dtype, torch.float32, seed=17, state=True, decay=8.0)
    k = x["k"].clone()
    if case == "one key":
        k[:] = k[:, :, :1]
    elif case == "two keys":
        k[:, :, ::2], k[:, :, 1::2] = k[:, :, :1], -k[:, :, 1:2]
    else:
        k = (k.float() * 0.05 + k[:, :, :1].float())
        k = (k / k.norm(dim=-1, keepdim=True)).to(dtype)
    x["k"] = k
    x["beta"][:] = beta
    grown = 1 + beta / (1 - abs(1 - beta))
    for name, a, b in zip(("o", "state", "dq", "dk", "dv", "dg", "dbeta", "ds0"), *run_both(x, 64)):
        err, norm = (a.detach().double() - b.detach()).norm().item(), b.detach().norm().item()
        assert err <= (tol(a.dtype) + (grown - 1) * F32_TOL) * norm, f"{name}: {err / norm:.3e}"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_long_training_sequence_of_wide_heads(dtype):
    x = make(1, 2, 1, 1700, 128, dtype, torch.bfloat16, seed=18, state=True, decay=6.0)
    compare(*run_both(x, 128))


def test_gradients_against_differences():
    """Directional derivatives of the library's own forward, through the fp32 state."""
    from simpletrain_b200 import gated_delta_chunk
    x = make(1, 2, 1, 100, 64, torch.float16, torch.float32, seed=5, state=True)
    gen = torch.Generator().manual_seed(9)
    for name in ("g", "beta", "s0"):  # fp32 inputs: they can be moved by a small step exactly
        d = torch.randn(x[name].shape, generator=gen).to(DEV)
        d = d / d.norm()
        leaf = x[name].detach().clone().requires_grad_(True)

        def loss(y):
            a = dict(x)
            a[name] = y
            _, s = gated_delta_chunk(*(a[n] for n in NAMES), initial_state=a["s0"])
            return (s.double() * x["dsT"].double()).sum()

        (grad,) = torch.autograd.grad(loss(leaf), leaf)
        # the state is smooth on the scale of 1: a central difference of step h is off by h^2 / 6 of a third
        # derivative of the same size as the first, plus 2^-17 |s| |ds| / h of the forward's own error
        h = 0.05
        with torch.no_grad():
            diff = (loss(x[name] + h * d) - loss(x[name] - h * d)) / (2 * h)
            size = gated_delta_chunk(*(x[n] for n in NAMES), initial_state=x["s0"])[1].norm() * x["dsT"].norm()
        allowed = h * h / 6 * 6 * grad.norm() + 2.0 ** -17 * size / h / 8
        assert (diff - (grad.double() * d.double()).sum()).abs() <= allowed, name


def test_second_derivatives_are_refused():
    from simpletrain_b200 import gated_delta_chunk
    from simpletrain_b200.fused_ops import token_logprobs
    x = make(1, 2, 1, 70, 64, torch.bfloat16, torch.float32, state=True)
    leaf = [x[n].requires_grad_(True) for n in NAMES]
    logits = torch.randn(3, 50, device=DEV, requires_grad=True)
    for out, wrt in ((gated_delta_chunk(*leaf, initial_state=x["s0"])[0].float().square().sum(), leaf),
                     (token_logprobs(logits, torch.zeros(3, dtype=torch.long, device=DEV)).logprob.square().sum(), [logits])):
        plain = torch.autograd.grad(out, wrt, retain_graph=True)
        again = torch.autograd.grad(out, wrt, create_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(plain, again))
        with pytest.raises(RuntimeError):  # the gradient is no function of the inputs
            torch.autograd.grad(again[0].float().sum(), wrt[0], retain_graph=True)
        with pytest.raises(RuntimeError, match="once"):
            again[0].float().sum().backward()


@pytest.mark.parametrize("T,B", [(0, 2), (5, 0)])
def test_empty(T, B):
    from simpletrain_b200 import gated_delta_chunk
    x = make(B, 2, 2, T, 64, torch.bfloat16, torch.float32, state=True)
    s0 = x["s0"].requires_grad_(True)
    leaf = [x[n].requires_grad_(True) for n in NAMES]
    o, s = gated_delta_chunk(*leaf, initial_state=s0)
    assert o.shape == (B, 2, T, 64) and torch.equal(s, s0)
    grads = torch.autograd.grad([o, s], leaf + [s0], [x["do"], x["dsT"]])
    assert torch.equal(grads[-1], x["dsT"]) and grads[0].shape == x["q"].shape
    cu = torch.zeros(1, dtype=torch.int32, device=DEV)  # no sequence at all
    if B == 2:
        y = make(1, 2, 2, 9, 64, torch.bfloat16, torch.float32)
        o, s = gated_delta_chunk(*(y[n] for n in NAMES), cu_seqlens=cu)
        assert (o == 0).all() and s.shape == (0, 2, 64, 64)


def test_long_sequence_and_state_handed_over():
    """A long stream, and the same stream in two calls with the state between them."""
    from simpletrain_b200 import gated_delta_chunk
    x = make(1, 2, 2, 5003, 64, torch.bfloat16, torch.float32, seed=6, decay=5.0)
    o, s = gated_delta_chunk(*(x[n] for n in NAMES))
    ref, s_ref = gated_delta(*(x[n].double() for n in NAMES), 64 ** -0.5)
    check("o", o, as_result(ref, o))
    check("s", s, as_result(s_ref, s))
    cut = 64 * 31
    o1, s1 = gated_delta_chunk(*(x[n][:, :, :cut] for n in NAMES))
    o2, s2 = gated_delta_chunk(*(x[n][:, :, cut:] for n in NAMES), initial_state=s1)
    assert torch.equal(torch.cat([o1, o2], 2), o) and torch.equal(s2, s)


def test_repeats_streams_and_capture():
    from simpletrain_b200 import gated_delta_chunk
    x = make(2, 4, 2, 200, 128, torch.bfloat16, torch.bfloat16, seed=7)
    y = make(2, 4, 2, 200, 128, torch.bfloat16, torch.bfloat16, seed=8)

    def step(z):
        leaf = [z[n].detach().requires_grad_(True) for n in NAMES]
        o, s = gated_delta_chunk(*leaf)
        return (o.detach(), s.detach(), *torch.autograd.grad(o, leaf, z["do"]))

    first, other = step(x), step(y)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(3):  # two calls at once
        for i, (st, z) in enumerate(zip(streams, (x, y))):
            with torch.cuda.stream(st):
                got[i] = step(z)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for z in (x, y):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(z))
        graphs.append(graph)
    for graph in graphs:  # replayed side by side
        with torch.cuda.stream(streams[graphs.index(graph)]):
            graph.replay()
    torch.cuda.synchronize()
    for want, a, b in zip((first, other), got, outs):
        for w, u, v in zip(want, a, b):
            assert torch.equal(w, u) and torch.equal(w, v)


def test_fp16_repeats_and_capture():
    """The units are found anew in every call: replays on other inputs, and a captured backward, give the eager bits."""
    from simpletrain_b200 import gated_delta_chunk
    cu, bounds, T = packed([150, 0, 64, 300])
    x, y = (make(1, 4, 2, T, 128, torch.float16, torch.float32, seed=s, state=True, n=4) for s in (23, 24))
    y = sized(y, v=50.0, s0=1e4, do=1e-4, dsT=1e-6)
    z = {n: t.detach().clone() for n, t in x.items()}

    def step(a):
        leaf = [a[n].detach().requires_grad_(True) for n in (*NAMES, "s0")]
        o, s = gated_delta_chunk(*leaf[:5], initial_state=leaf[5], cu_seqlens=cu)
        return (o.detach(), s.detach(), *torch.autograd.grad([o, s], leaf, [a["do"], a["dsT"]]))

    want = [[t.clone() for t in step(a)] for a in (x, y, x)]
    assert all(torch.equal(a, b) for a, b in zip(want[0], want[2]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(z)
    for a, w in ((x, want[0]), (y, want[1]), (x, want[0])):
        for n in z:
            z[n].copy_(a[n])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(w, out))


def test_compiled_calls():
    """Traced with fake tensors, forward and backward, the ops are called as they are in eager mode."""
    from simpletrain_b200 import gated_delta_chunk, gated_delta_step
    from simpletrain_b200.fused_ops import token_logprobs
    x = make(2, 4, 2, 130, 64, torch.bfloat16, torch.float32, state=True)
    head = torch.randn(64, 50, device=DEV, dtype=torch.bfloat16)
    tok = torch.arange(2 * 4 * 130, device=DEV) % 50
    leaf = [x[n].detach().requires_grad_(True) for n in (*NAMES, "s0")]

    def loss(*a):
        o, s = gated_delta_chunk(*a[:5], initial_state=a[5])
        r = token_logprobs((o @ head).reshape(-1, 50), tok, top_k=2)
        return r.logprob.mean() + 0.1 * r.entropy.mean() + s.square().mean()

    a = step_inputs(3, 2, 1, 64, 5, torch.bfloat16)
    states = [a["state"].clone() for _ in range(2)]
    results = []
    for i, wrap in enumerate((lambda f: f, lambda f: torch.compile(f, backend="aot_eager", fullgraph=True))):
        got = wrap(loss)(*leaf)
        with torch.no_grad():
            o = wrap(lambda *t: gated_delta_step(*t) * 2)(*(a[n] for n in NAMES), states[i])
        results.append((got.detach(), *torch.autograd.grad(got, leaf), o, states[i]))
    assert all(torch.equal(u, v) for u, v in zip(*results))


# ------------------------------------------------------------------- step --
def step_inputs(N, H, Hk, D, states, dtype, gate=torch.float32, seed=0):
    x = make(1, H, Hk, N, D, dtype, gate, seed=seed)
    a = {n: x[n][0].transpose(0, 1) for n in NAMES}  # [N, heads, ...] views
    gen = torch.Generator().manual_seed(seed + 100)
    a["state"] = (0.3 * torch.randn(states, H, D, D, generator=gen)).to(DEV)
    return a


def step_ref(a, slots, scale, rows=None):
    """float64, rows in order."""
    H, Hk = a["v"].shape[1], a["q"].shape[1]
    st = a["state"].double().clone()
    o = torch.zeros(a["v"].shape, dtype=torch.float64, device=DEV)
    for n, s in enumerate(slots):
        if 0 <= s < st.shape[0]:
            q, k = (a[m][n].double().repeat_interleave(H // Hk, 0) for m in "qk")
            S = st[s] * a["g"][n].double().exp()[:, None, None]
            u = a["beta"][n].double()[:, None] * (a["v"][n].double() - torch.einsum("hkv,hk->hv", S, k))
            S = S + k[:, :, None] * u[:, None]
            st[s], o[n] = S, scale * torch.einsum("hkv,hk->hv", S, q)
    return o, st


@pytest.mark.parametrize("N,H,Hk,D,states,dtype,gate,slots", [
    (1, 1, 1, 64, 1, torch.bfloat16, torch.float32, None),
    (3, 4, 2, 128, 5, torch.bfloat16, torch.bfloat16, None),
    (5, 2, 2, 128, 7, torch.float16, torch.float32, [6, 0, 3, 2, 5]),
    (7, 3, 1, 64, 4, torch.bfloat16, torch.float16, [2, -1, 2, 0, 2, -7, 0]),   # the same state more than once, padding
    (300, 2, 1, 64, 12, torch.bfloat16, torch.float32, [(7 * i) % 13 - 1 for i in range(300)]),
])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_step(N, H, Hk, D, states, dtype, gate, slots, index):
    from simpletrain_b200 import device_status, gated_delta_step
    a = step_inputs(N, H, Hk, D, states, dtype, gate)
    idx = None if slots is None else torch.tensor(slots, dtype=index, device=DEV)
    o_ref, s_ref = step_ref(a, range(N) if slots is None else slots, D ** -0.5)
    before = a["state"].clone()
    o = gated_delta_step(a["q"], a["k"], a["v"], a["g"], a["beta"], a["state"], state_indices=idx)
    assert device_status() == 0
    check("o", o, as_result(o_ref, o))
    check("state", a["state"], as_result(s_ref, a["state"]))
    used = set(range(N) if slots is None else slots)
    for s in set(range(states)) - used:
        assert torch.equal(a["state"][s], before[s])


def test_inference_mode_and_in_place_counting():
    """Inference tensors are taken; an ordinary pool's version moves with every step, so a graph that saved it notices."""
    from simpletrain_b200 import gated_delta_chunk, gated_delta_step
    a = step_inputs(3, 2, 1, 64, 4, torch.bfloat16)
    want = a["state"].clone()
    o = gated_delta_step(*(a[n] for n in NAMES), want)
    with torch.inference_mode():
        b = {n: t.clone() for n, t in a.items()}
        assert torch.equal(gated_delta_step(*(b[n] for n in NAMES), b["state"]), o) and torch.equal(b["state"], want)
        x = [b[n].transpose(0, 1)[None] for n in NAMES]
        assert gated_delta_chunk(*x)[0].shape == (1, 2, 3, 64)
    w = torch.ones(4, 2, 64, 64, device=DEV, requires_grad=True)
    loss = (w * a["state"]).sum()
    gated_delta_step(*(a[n] for n in NAMES), a["state"])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_step_on_a_strided_pool_and_bad_indices():
    from simpletrain_b200 import _ffi, device_status, gated_delta_step
    a = step_inputs(4, 2, 2, 64, 6, torch.bfloat16)
    layers = torch.randn(6, 3, 2, 64, 64, generator=torch.Generator().manual_seed(1)).to(DEV)  # [slot, layer, H, D, D]
    keep = layers.clone()
    a["state"] = layers[:, 1]
    slots = [4, 6, 1, 2 ** 33]  # two of them name no state
    o_ref, s_ref = step_ref(a, slots, 0.5)
    o = gated_delta_step(a["q"], a["k"], a["v"], a["g"], a["beta"], layers[:, 1], scale=0.5,
                         state_indices=torch.tensor(slots, device=DEV))
    assert device_status() == _ffi.KDA_ERR_DEVICE_INDEX
    check("o", o, as_result(o_ref, o))
    check("state", layers[:, 1], as_result(s_ref, layers))
    assert torch.equal(layers[:, 0], keep[:, 0]) and torch.equal(layers[:, 2], keep[:, 2])
    assert (o[1] == 0).all() and (o[3] == 0).all()
    with pytest.raises(RuntimeError):  # one state for all rows cannot be updated in place
        gated_delta_step(a["q"], a["k"], a["v"], a["g"], a["beta"], layers[:1, 0].expand(4, 2, 64, 64))
    flat = torch.zeros(9 * 64 * 64, device=DEV)
    with pytest.raises(RuntimeError, match="apart"):  # head 1 of a state is head 0 of the next
        gated_delta_step(a["q"], a["k"], a["v"], a["g"], a["beta"], flat.as_strided((6, 2, 64, 64), (4096, 4096, 64, 1)))
    by_head = flat[:2 * 4 * 4096].view(2, 4, 64, 64).transpose(0, 1)  # [heads, states] memory
    assert gated_delta_step(a["q"], a["k"], a["v"], a["g"], a["beta"], by_head).shape == (4, 2, 64)


def test_step_on_every_third_head_of_a_pool():
    """States need only be apart: a slice of another model's heads is taken as it is."""
    from simpletrain_b200 import gated_delta_step
    a = step_inputs(3, 4, 2, 64, 5, torch.bfloat16)
    wide = torch.randn(5, 10, 64, 64, generator=torch.Generator().manual_seed(2)).to(DEV)
    keep = wide.clone()
    a["state"] = wide[:, ::3]
    o_ref, s_ref = step_ref(a, [4, 1, 0], 64 ** -0.5)
    o = gated_delta_step(*(a[n] for n in NAMES), wide[:, ::3], state_indices=torch.tensor([4, 1, 0], device=DEV))
    check("o", o, as_result(o_ref, o))
    check("state", wide[:, ::3], as_result(s_ref, wide))
    for h in (1, 2, 4, 5, 7, 8):
        assert torch.equal(wide[:, h], keep[:, h])


@pytest.mark.parametrize("layout", ["heads first", "tokens first", "fused", "broadcast"])
def test_fake_implementations_tell_the_truth(layout):
    """Shapes, strides and types of the ops under fake tensors are those of the real ones (what a compiler builds on)."""
    from simpletrain_b200 import delta, fused_ops  # noqa: F401  (register them)
    from torch._subclasses.fake_tensor import FakeTensorMode
    B, H, T, D = 2, 4, 70, 64
    x = make(B, H, H, T, D, torch.bfloat16, torch.float32, state=True)
    a = {n: x[n].contiguous() if layout == "heads first" else x[n] for n in (*NAMES, "do")}
    if layout == "fused":
        proj = torch.stack([x[n].transpose(1, 2) for n in "qkv"], 2)
        a.update(zip("qkv", (t.transpose(1, 2) for t in proj.unbind(2))))
    if layout == "broadcast":
        a["k"] = a["k"][:, :1].expand(B, H, T, D)
        a["v"] = a["v"][:1].expand(B, H, T, D)
    logits = torch.randn(5, 40, device=DEV)[:, :33]
    row = torch.zeros(5, device=DEV)
    st = {n: a[n][:, :, 0] for n in NAMES}
    ops = torch.ops.kda_b200
    calls = [
        lambda t: ops.delta_fwd(*(t[n] for n in NAMES), 0.1, t["s0"], None, True),
        lambda t: ops.delta_fwd(*(t[n] for n in NAMES), 0.1, None, None, False),
        lambda t: ops.delta_bwd(*(t[n] for n in NAMES), 0.1, t["s0"], None, t["do"], None, True),
        lambda t: (ops.delta_step(*(t["st_" + n] for n in NAMES), t["s0"], None, 0.1),),
        lambda t: torch.ops.st_b200.token_logprobs(t["logits"], t["tok"], 3, 1.0, -100),
    ]
    real = {**a, "s0": x["s0"], "logits": logits, "tok": row.long(), **{"st_" + n: t for n, t in st.items()}}
    with FakeTensorMode() as mode:
        fake = {n: mode.from_tensor(t) for n, t in real.items()}
        told = [call(fake) for call in calls]
    for call, said in zip(calls, told):
        for r, f in zip(call(real), said):
            assert r.shape == f.shape and r.dtype == f.dtype and r.device == f.device
            assert r.numel() == 0 or [s for s, n in zip(r.stride(), r.shape) if n > 1] == [s for s, n in zip(f.stride(), f.shape) if n > 1]


def test_offsets_past_32_bits():
    """The last head of a long call and the last states of a large pool are what they are on their own."""
    from simpletrain_b200 import gated_delta_chunk, gated_delta_step
    H, T, D = 33, 1 << 20, 64
    gen = torch.Generator(device=DEV).manual_seed(22)

    def rnd(*shape):
        return torch.randn(*shape, generator=gen, device=DEV, dtype=torch.bfloat16)

    v = rnd(1, H, T, D)
    assert v.numel() > 1 << 31
    k = torch.nn.functional.normalize(rnd(1, 1, T, D), dim=-1)
    q = k.flip(2)
    g, beta = -torch.rand(1, H, T, generator=gen, device=DEV), torch.rand(1, H, T, generator=gen, device=DEV)
    o, s = gated_delta_chunk(q, k, v, g, beta)
    oi, si = gated_delta_chunk(q, k, v[:, -1:], g[:, -1:], beta[:, -1:])
    assert torch.equal(o[:, -1:], oi) and torch.equal(s[:, -1:], si)
    del o, v
    pool = torch.zeros((1 << 31) // (2 * D * D) + 3, 2, D, D, device=DEV)
    assert pool[-1].storage_offset() > 1 << 31
    a = step_inputs(2, 2, 1, D, 3, torch.bfloat16)
    n = pool.shape[0]
    pool[-1], pool[-3] = a["state"][0], a["state"][1]
    o1 = gated_delta_step(*(a[m] for m in NAMES), a["state"])
    o2 = gated_delta_step(*(a[m] for m in NAMES), pool, state_indices=torch.tensor([n - 1, n - 3], device=DEV))
    assert torch.equal(o1, o2) and torch.equal(pool[-1], a["state"][0]) and torch.equal(pool[-3], a["state"][1])
    assert not pool[0].any() and not pool[-2].any()


def test_prefill_steps_and_scores_agree():
    """Prefill, single steps with the tokens' log probabilities, and the chunked form over the whole
    sequence with its gradient: the three operators as a serving and a training loop use them."""
    from simpletrain_b200 import gated_delta_chunk, gated_delta_step
    from simpletrain_b200.fused_ops import token_logprobs
    B, H, T, D, V, cut = 3, 2, 90, 64, 211, 70
    x = make(B, H, 1, T, D, torch.bfloat16, torch.float32, seed=11)
    gen = torch.Generator().manual_seed(12)
    head = (torch.randn(H * D, V, generator=gen) * 0.2).to(torch.bfloat16).to(DEV)
    tok = torch.randint(0, V, (B, T), generator=gen).to(DEV)
    leaf = [x[n].detach().requires_grad_(True) for n in NAMES]
    o, _ = gated_delta_chunk(*leaf)
    logits = o.transpose(1, 2).reshape(B * T, H * D) @ head
    score = token_logprobs(logits, tok.view(-1), top_k=4, temperature=0.8)
    grads = torch.autograd.grad(score.logprob.mean() + 0.01 * score.entropy.mean(), leaf)
    pool = torch.zeros(5, H, D, D, device=DEV)
    slots = torch.tensor([4, 0, 2], device=DEV)
    with torch.no_grad():
        _, s = gated_delta_chunk(*(x[n][:, :, :cut] for n in NAMES))
        pool[slots] = s
        for t in range(cut, T):
            ot = gated_delta_step(*(x[n][:, :, t] for n in NAMES), pool, state_indices=slots)
            # chunked and stepped o differ by a rounding of the 16-bit output each at most
            want = o[:, :, t]
            assert (ot.double() - want.double()).norm() <= 2 * tol(torch.bfloat16) * want.double().norm()
            r = token_logprobs(ot.reshape(B, H * D) @ head, tok[:, t], top_k=4, temperature=0.8)
            full = score.logprob.view(B, T)[:, t]
            # logits: a sum of H D products, o and the head's result each off by half a bf16 step
            size = (ot.reshape(B, H * D).float().norm(dim=1) * head.float().norm(dim=0).max()).max().item()
            assert (r.logprob - full).abs().max() <= 2 * 3 * 2.0 ** -8 * size / 0.8
    # the gradients against the definitions in float64, from the same logits' gradient
    ref = [x[n].double().requires_grad_(True) for n in NAMES]
    o64, _ = gated_delta(*ref, D ** -0.5)
    again = logits.detach().requires_grad_(True)
    r = token_logprobs(again, tok.view(-1), temperature=0.8)
    (dlogits,) = torch.autograd.grad(r.logprob.mean() + 0.01 * r.entropy.mean(), again)
    do = (dlogits @ head.t()).view(B, T, H, D).transpose(1, 2)
    want = torch.autograd.grad(o64, ref, do.double())
    for n, a, b in zip(NAMES, grads, want):
        check(n, a, as_result(b, a))
