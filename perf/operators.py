"""Cases for the gated delta rule (chunked scan, its gradients, the single-token
step over a pool of states) and for the log probabilities of given tokens.

``own`` false: plain torch in 32 bits.  ``own`` true: the calls a user makes of
``simpletrain_b200``.  Shapes are those of the scan's model variants (100m: 8
heads of 64; 1b: 10 heads of 128; 7b: 24 heads of 128; 10b: 28 heads of 128; a
vocabulary of 32000) and odd sizes between them.

Formulas.  Per (sequence, head), with S the [D, D] state (row = key channel):

    S' = exp(g_t) S_{t-1}         u_t = beta_t (v_t - S'^T k_t)
    S_t = S' + k_t u_t^T          o_t = scale * S_t^T q_t

Log probabilities, x = logits / temperature, p = softmax(x):

    logprob = x_token - lse(x)    entropy = lse(x) - sum_v p_v x_v
"""
import math

import torch

own = False

CHUNK = 64
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------- cases --
def listed():
    return [
        # a training step's scan at the 1b variant's micro-batch: forward and all gradients
        {"name": "delta train 1b", "op": "train", "B": 16, "T": 2048, "H": 10, "Hk": 10, "D": 128, "packed": 0, "dtype": "bf16"},
        # documents packed into one row with offsets, query/key heads shared by two value heads, D = 64
        {"name": "delta train packed", "op": "train", "B": 1, "T": 16349, "H": 8, "Hk": 4, "D": 64, "packed": 23, "dtype": "bf16"},
        # a small fine-tuning batch of odd length, fp16
        {"name": "delta train small", "op": "train", "B": 2, "T": 333, "H": 8, "Hk": 8, "D": 64, "packed": 0, "dtype": "fp16"},
        # prefill of one long context at the 10b variant, resumed from a state
        {"name": "delta prefill long", "op": "prefill", "B": 1, "T": 32768, "H": 28, "Hk": 28, "D": 128, "packed": 0, "dtype": "bf16"},
        # prefill of one short odd prompt: latency counts
        {"name": "delta prefill short", "op": "prefill", "B": 1, "T": 177, "H": 10, "Hk": 10, "D": 128, "packed": 0, "dtype": "bf16"},
        # one new token for one user, 100m variant: the smallest call
        {"name": "delta step 1", "op": "step", "N": 1, "slots": 4, "H": 8, "Hk": 8, "D": 64, "dtype": "bf16"},
        # one new token for a small odd batch, grouped heads
        {"name": "delta step 37", "op": "step", "N": 37, "slots": 48, "H": 24, "Hk": 8, "D": 128, "dtype": "fp16"},
        # one new token each for a full serving batch, 10b variant
        {"name": "delta step 256", "op": "step", "N": 256, "slots": 256, "H": 28, "Hk": 28, "D": 128, "dtype": "bf16"},
        # log probability and 5 alternatives of one sampled token
        {"name": "logprobs serve 1", "op": "score", "N": 1, "V": 32000, "k": 5, "temperature": 1.0, "dtype": "bf16"},
        # the same for a serving batch whose head gives fp32 logits, odd vocabulary, sampling temperature
        {"name": "logprobs serve 128", "op": "score", "N": 128, "V": 50257, "k": 20, "temperature": 0.7, "dtype": "fp32"},
        # log probabilities and entropies of a micro-batch, with the logits' gradient (policy-gradient step)
        {"name": "logprobs train", "op": "logtrain", "N": 16384, "V": 32000, "temperature": 1.0, "dtype": "bf16"},
        # the same, small, odd vocabulary
        {"name": "logprobs train odd", "op": "logtrain", "N": 1021, "V": 10007, "temperature": 0.8, "dtype": "fp16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["train", "train", "prefill", "step", "score", "logtrain"])
    if op in ("train", "prefill"):
        D = rng.choice([64, 128])
        H = rng.choice([2, 4, 8, 10, 12, 16])
        Hk = H // rng.choice([1, 1, 2])
        packed = rng.choice([0, 0, rng.randint(2, 40)])
        B = 1 if packed else rng.randint(1, 8)
        T = _log(rng, 65, 4096) if op == "train" else _log(rng, 1, 8192)
        return {"op": op, "B": B, "T": T, "H": H, "Hk": Hk, "D": D, "packed": packed, "dtype": rng.choice(["bf16", "bf16", "fp16"])}
    if op == "step":
        N = _log(rng, 1, 200)
        H = rng.choice([4, 8, 10, 24])
        return {"op": op, "N": N, "slots": N + rng.randint(0, 40), "H": H, "Hk": H // rng.choice([1, 2]), "D": rng.choice([64, 128]),
                "dtype": rng.choice(["bf16", "fp16"])}
    V = _log(rng, 1000, 130000)
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    t = rng.choice([1.0, 0.7, 1.3])
    if op == "score":
        return {"op": op, "N": _log(rng, 1, 300), "V": V, "k": rng.randint(1, 32), "temperature": t, "dtype": dtype}
    return {"op": op, "N": max(1, _log(rng, 1000, 200_000_000) // V), "V": V, "temperature": t, "dtype": dtype}


# ----------------------------------------------------------------- prepare --
def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dt = DT[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    def unit(*shape):  # q, k: L2-normalised over the head dimension
        x = normal(*shape)
        return (x / x.norm(dim=-1, keepdim=True)).to(dt)

    s = dict(case)
    if case["op"] in ("train", "prefill"):
        B, T, H, Hk, D = (case[n] for n in ("B", "T", "H", "Hk", "D"))
        train = case["op"] == "train"
        # [B, H, T, D] views over [B, T, H, D] memory, as a layer's projections give them
        s["q"], s["k"] = unit(B, T, Hk, D).transpose(1, 2), unit(B, T, Hk, D).transpose(1, 2)
        s["v"] = normal(B, T, H, D).to(dt).transpose(1, 2)
        # log decay and write strength: projections of the model's type when training, fp32 when serving
        gt = dt if train else torch.float32
        s["g"] = torch.nn.functional.logsigmoid(normal(B, T, H) + 3.0).to(gt).transpose(1, 2)
        s["beta"] = torch.sigmoid(normal(B, T, H)).to(gt).transpose(1, 2)
        n = B
        s["cu"] = None
        if case["packed"]:
            n = case["packed"]
            cuts = torch.randint(0, T + 1, (n - 1,), generator=gen, device=dev, dtype=torch.int32).sort().values
            ends = torch.tensor([0, T], device=dev, dtype=torch.int32)
            s["cu"] = torch.cat([ends[:1], cuts, ends[1:]])
        s["s0"] = None if train else normal(n, H, D, D) * 0.1
        if train:
            s["do"] = normal(B, T, H, D).to(dt).transpose(1, 2)
            for name in ("q", "k", "v", "g", "beta"):
                s[name].requires_grad_(True)
    elif case["op"] == "step":
        N, H, Hk, D = (case[n] for n in ("N", "H", "Hk", "D"))
        s["q"], s["k"], s["v"] = unit(N, Hk, D), unit(N, Hk, D), normal(N, H, D).to(dt)
        s["g"] = torch.nn.functional.logsigmoid(normal(N, H) + 3.0)
        s["beta"] = torch.sigmoid(normal(N, H))
        s["state"] = normal(case["slots"], H, D, D) * 0.3
        s["slot"] = torch.randperm(case["slots"], generator=gen, device=dev)[:N].to(torch.int32)
    else:
        N, V = case["N"], case["V"]
        x = torch.empty(N, V, device=dev, dtype=dt).normal_(0.0, 3.0, generator=gen)
        s["tokens"] = torch.randint(0, V, (N,), generator=gen, device=dev)
        s["logits"] = x
        if case["op"] == "logtrain":
            x.requires_grad_(True)
            s["dlogprob"], s["dentropy"] = normal(N) / N, normal(N) * (0.01 / N)
    return s


# ------------------------------------------------------------- plain forms --
def _inverse(A):
    """(I + A)^-1 of strictly lower triangular [..., n, n] matrices, n a power of two, by halves."""
    n = A.shape[-1]
    if n == 1:
        return torch.ones_like(A)
    h = n // 2
    a, c = _inverse(A[..., :h, :h]), _inverse(A[..., h:, h:])
    off = -(c @ A[..., h:, :h] @ a)
    return torch.cat([torch.cat([a, torch.zeros_like(off)], -1), torch.cat([off, c], -1)], -2)


def _gather(s, names):
    """[n, H, C * chunks, ...] fp32 tensors with one sequence a row, zero behind each sequence's end, and where the rows came from."""
    T = s["T"]
    if s["cu"] is None:
        idx = torch.arange(T, device="cuda")[None]
        live = torch.ones_like(idx, dtype=torch.bool)
    else:
        cu = s["cu"].long()
        most = int((cu[1:] - cu[:-1]).max())
        idx = cu[:-1, None] + torch.arange(most, device="cuda")
        live = idx < cu[1:, None]
    pad = -idx.shape[1] % CHUNK
    idx, live = (torch.nn.functional.pad(x, (0, pad)) for x in (idx, live))
    at = torch.where(live, idx, 0)
    out = []
    for name in names:
        x = s[name].float()
        G = s["H"] // x.shape[1]
        x = x.repeat_interleave(G, 1)
        x = x[:, :, at[0]] if s["cu"] is None else x[0][:, at].transpose(0, 1)
        m = live[:, None] if x.dim() == 3 else live[:, None, :, None]
        out.append(torch.where(m, x, 0.0))
    return out, idx, live


def _plain_scan(s):
    (q, k, v, g, beta), idx, live = _gather(s, ("q", "k", "v", "g", "beta"))
    D, T = s["D"], s["T"]
    n, H, L = g.shape
    scale = D ** -0.5

    def chunked(x):
        return x.reshape(n, H, L // CHUNK, CHUNK, *x.shape[3:])

    q, k, v, g, beta = map(chunked, (q, k, v, g, beta))
    gam = g.double().cumsum(-1)
    keep = torch.ones(CHUNK, CHUNK, device="cuda", dtype=torch.bool).tril()
    dec = torch.where(keep, gam[..., :, None] - gam[..., None, :], -math.inf).exp().float()
    A = (beta[..., None] * dec * (k @ k.mT)).tril(-1)
    P = scale * dec * (q @ k.mT)
    inv = _inverse(A)
    G = gam.exp().float()[..., None]
    last = gam[..., -1:].exp().float()[..., None]
    left = (gam[..., -1:] - gam).exp().float()[..., None]
    S = s["s0"] if s["s0"] is not None else torch.zeros(n, H, D, D, device="cuda")
    o = []
    for c in range(L // CHUNK):  # the state passes from chunk to chunk
        K, Q = k[:, :, c], q[:, :, c]
        u = inv[:, :, c] @ (beta[:, :, c, :, None] * (v[:, :, c] - G[:, :, c] * (K @ S)))
        o.append(scale * G[:, :, c] * (Q @ S) + P[:, :, c] @ u)
        S = last[:, :, c] * S + K.mT @ (left[:, :, c] * u)
    o = torch.stack(o, 2).reshape(n, H, L, D)
    if s["cu"] is None:
        o = o[:, :, :T]
    else:
        o = o.transpose(0, 1)[:, live][None]  # the sequences' rows in their order are all rows
    return o.to(s["v"].dtype), S


def _plain_step(s):
    q, k, v = (s[n].float() for n in ("q", "k", "v"))
    G = s["H"] // s["Hk"]
    q, k = q.repeat_interleave(G, 1), k.repeat_interleave(G, 1)
    slot = s["slot"].long()
    S = s["state"][slot] * s["g"].exp()[..., None, None]
    u = s["beta"][..., None] * (v - (S * k[..., :, None]).sum(-2))
    S = S + k[..., :, None] * u[..., None, :]
    o = s["D"] ** -0.5 * (S * q[..., :, None]).sum(-2)
    s["state"][slot] = S
    return o.to(s["v"].dtype), s["state"]


def _plain_logprobs(s, top):
    x = s["logits"].float() / s["temperature"]
    m = x.detach().amax(-1, keepdim=True)
    e = (x - m).exp()
    z = e.sum(-1)
    lse = m[:, 0] + z.log()
    lp = x.gather(1, s["tokens"][:, None])[:, 0] - lse
    H = z.log() - (e * (x - m)).sum(-1) / z
    if not top:
        return lp, H
    ids = s["logits"].sort(dim=-1, descending=True, stable=True).indices[:, :top]  # ties: the lowest index first
    return lp, H, x.gather(1, ids) - lse[:, None], ids


# --------------------------------------------------------------------- run --
def run(state):
    s, op = state, state["op"]
    if op in ("train", "prefill"):
        if own:
            from simpletrain_b200 import gated_delta_chunk
            o, S = gated_delta_chunk(s["q"], s["k"], s["v"], s["g"], s["beta"], initial_state=s["s0"], cu_seqlens=s["cu"],
                                     output_final_state=op == "prefill")
        else:
            o, S = _plain_scan(s)
        if op == "prefill":
            return o, S
        return (o.detach(),) + torch.autograd.grad(o, [s[n] for n in ("q", "k", "v", "g", "beta")], s["do"])
    if op == "step":
        if own:
            from simpletrain_b200 import gated_delta_step
            o = gated_delta_step(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"], state_indices=s["slot"])
            return o, s["state"]
        return _plain_step(s)
    if own:
        from simpletrain_b200.fused_ops import token_logprobs
        r = token_logprobs(s["logits"], s["tokens"], top_k=s.get("k", 0), temperature=s["temperature"])
        r = (r.logprob, r.entropy) if op == "logtrain" else (r.logprob, r.entropy, r.top_logprobs, r.top_ids)
    else:
        r = _plain_logprobs(s, s.get("k", 0))
    if op == "score":
        return r
    (dx,) = torch.autograd.grad(r, [s["logits"]], (s["dlogprob"], s["dentropy"]))
    return r[0].detach(), r[1].detach(), dx


# -------------------------------------------------------------------- work --
def work(case):
    op = case["op"]
    w = 4 if case["dtype"] == "fp32" else 2
    if op in ("train", "prefill"):
        B, T, H, Hk, D = (case[n] for n in ("B", "T", "H", "Hk", "D"))
        rows = B * T
        heads = (2 * Hk + 2 * H) * D * 2  # q, k, v in and o out, a token
        n = case["packed"] or B
        if op == "prefill":
            return {"bytes": rows * (heads + 8 * H) + 8 * n * H * D * D, "flops": rows * H * 6 * D * D}
        # forward, then q, k, v, gates and do in, five gradients out; the recurrence's products and twice those backward
        return {"bytes": rows * (heads + 4 * H + (4 * Hk + 3 * H) * D * 2 + 8 * H), "flops": rows * H * 18 * D * D}
    if op == "step":
        N, H, Hk, D = (case[n] for n in ("N", "H", "Hk", "D"))
        return {"bytes": N * (8 * H * D * D + 4 * (Hk + H) * D + 8 * H + 4), "flops": N * H * 7 * D * D}
    N, V = case["N"], case["V"]
    if op == "score":
        return {"bytes": N * (V * w + 16 + 12 * case["k"]), "flops": 5 * N * V}
    # the logits are needed twice (the row's sum comes before its gradient), the gradient is written
    return {"bytes": N * (3 * V * w + 24), "flops": 12 * N * V}


# ------------------------------------------------------- the definition in 64 bits --
def _tokens(q, k, v, g, beta, S, scale):
    """The recurrence, token by token: [R, t, ...] inputs, [R, D, D] state."""
    o = []
    for t in range(q.shape[1]):
        S = S * g[:, t, None, None].exp()
        u = beta[:, t, None] * (v[:, t] - torch.einsum("rkv,rk->rv", S, k[:, t]))
        S = S + torch.einsum("rk,rv->rkv", k[:, t], u)
        o.append(torch.einsum("rkv,rk->rv", S, q[:, t]) * scale)
    return torch.stack(o, 1), S


def _exact_scan(s, train):
    d = torch.float64
    B, T, H, D = s["B"], s["T"], s["H"], s["D"]
    G = H // s["Hk"]
    bounds = [(b, 0, T) for b in range(B)] if s["cu"] is None else \
        [(0, lo, hi) for lo, hi in zip(s["cu"].tolist()[:-1], s["cu"].tolist()[1:])]
    most = max(hi - lo for _, lo, hi in bounds)
    names = ("q", "k", "v", "g", "beta") + (("do",) if train else ())
    x = {}
    for name in names:  # one row a (sequence, head); behind the end: g = beta = 0 and zeros, which change nothing
        src = s[name].detach().to(d)
        src = src.repeat_interleave(H // src.shape[1], 1)
        y = torch.zeros(len(bounds), H, most, *src.shape[3:], device="cuda", dtype=d)
        for i, (b, lo, hi) in enumerate(bounds):
            y[i, :, : hi - lo] = src[b, :, lo:hi]
        x[name] = y.reshape(len(bounds) * H, most, *src.shape[3:])
    R = len(bounds) * H
    S = torch.zeros(R, D, D, device="cuda", dtype=d) if s["s0"] is None else s["s0"].to(d).reshape(R, D, D)
    scale = D ** -0.5
    step = 32
    states, outs = [], []
    with torch.no_grad():
        for t in range(0, most, step):
            states.append(S if train else None)
            o, S = _tokens(*(x[n][:, t:t + step] for n in names[:5]), S, scale)
            outs.append(o)

    def back(y, like):
        y = y.reshape(len(bounds), H, most, *y.shape[2:])
        z = torch.zeros(B, H, T, *y.shape[3:], device="cuda", dtype=d)
        for i, (b, lo, hi) in enumerate(bounds):
            z[b, :, lo:hi] = y[i, :, : hi - lo]
        return z.reshape(B, like.shape[1], H // like.shape[1], *z.shape[2:]).sum(2)

    o = back(torch.cat(outs, 1), s["v"])
    if not train:
        return o, S.reshape(len(bounds), H, D, D)
    grads = {n: [] for n in names[:5]}
    dS = torch.zeros_like(S)
    for i in reversed(range(len(states))):  # gradients by spans of tokens, from each span's first state
        t = i * step
        leaves = [x[n][:, t:t + step].clone().requires_grad_(True) for n in names[:5]]
        S0 = states[i].clone().requires_grad_(True)
        o_, S_ = _tokens(*leaves, S0, scale)
        got = torch.autograd.grad([o_, S_], leaves + [S0], [x["do"][:, t:t + step], dS])
        dS = got[5]
        for n, y in zip(names[:5], got):
            grads[n].append(y)
    return (o,) + tuple(back(torch.cat(grads[n][::-1], 1), s[n]) for n in names[:5])


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("train", "prefill"):
        return _exact_scan(s, op == "train")
    d = torch.float64
    if op == "step":
        G = case["H"] // case["Hk"]
        q, k, v = s["q"].to(d), s["k"].to(d), s["v"].to(d)
        pool = s["state"].to(d)
        o = torch.zeros_like(v)
        for h in range(case["H"]):
            S = pool[s["slot"].long(), h] * s["g"][:, h].to(d).exp()[:, None, None]
            kh, qh = k[:, h // G], q[:, h // G]
            u = s["beta"][:, h].to(d)[:, None] * (v[:, h] - torch.einsum("nkv,nk->nv", S, kh))
            S = S + torch.einsum("nk,nv->nkv", kh, u)
            pool[s["slot"].long(), h] = S
            o[:, h] = torch.einsum("nkv,nk->nv", S, qh) * case["D"] ** -0.5
        return o, pool
    parts = []
    rows = max(1, 50_000_000 // case["V"])
    for r in range(0, case["N"], rows):
        x = s["logits"][r:r + rows].detach().to(d) / case["temperature"]
        tok = s["tokens"][r:r + rows, None]
        lp = torch.log_softmax(x, -1)
        p = lp.exp()
        H = -(p * lp).sum(-1)
        if op == "score":
            ids = torch.sort(s["logits"][r:r + rows], dim=-1, descending=True, stable=True).indices[:, :case["k"]]
            parts.append((lp.gather(1, tok)[:, 0], H, lp.gather(1, ids), ids))
        else:
            a, b = s["dlogprob"][r:r + rows, None].to(d), s["dentropy"][r:r + rows, None].to(d)
            dx = -p * a - b * p * (lp + H[:, None])
            dx.scatter_add_(1, tok, a)
            parts.append((lp.gather(1, tok)[:, 0], H, (dx / case["temperature"]).to(torch.float32)))
    return tuple(torch.cat(c) for c in zip(*parts))
