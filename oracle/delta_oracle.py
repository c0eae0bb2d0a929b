"""The gated delta rule and token log probabilities from their definitions, in float64.

Plain torch, any device, differentiable; nothing of the library is used.
"""
from __future__ import annotations

import torch


def delta_recurrence(q, k, v, g, beta, scale, state=None):
    """Token by token: q, k [H, T, D], v [H, T, D], g, beta [H, T], state [H, D, D] -> (o, state)."""
    H, T, D = v.shape
    S = torch.zeros(H, D, D, dtype=v.dtype, device=v.device) if state is None else state
    o = []
    for t in range(T):
        S = S * g[:, t, None, None].exp()
        u = beta[:, t, None] * (v[:, t] - torch.einsum("hkv,hk->hv", S, k[:, t]))
        S = S + k[:, t, :, None] * u[:, None, :]
        o.append(scale * torch.einsum("hkv,hk->hv", S, q[:, t]))
    return (torch.stack(o, 1) if T else v * 1), S


def gated_delta(q, k, v, g, beta, scale, state=None, bounds=None):
    """[B, Hk, T, D] / [B, H, T, ...] inputs as the library takes them; ``bounds``: (start, end) of
    the sequences packed into a batch of one.  Returns (o [B, H, T, D], final states)."""
    B, H, T, D = v.shape
    G = H // q.shape[1]
    q, k = q.repeat_interleave(G, 1), k.repeat_interleave(G, 1)
    spans = [(b, 0, T) for b in range(B)] if bounds is None else [(0, lo, hi) for lo, hi in bounds]
    o = torch.zeros_like(v)
    states = []
    for i, (b, lo, hi) in enumerate(spans):
        S0 = None if state is None else state[i]
        oi, S = delta_recurrence(q[b, :, lo:hi], k[b, :, lo:hi], v[b, :, lo:hi], g[b, :, lo:hi], beta[b, :, lo:hi], scale, S0)
        o = torch.cat([o[:, :, :lo], oi[None], o[:, :, hi:]], 2) if bounds is not None else \
            torch.cat([o[:b], oi[None], o[b + 1:]], 0)
        states.append(S)
    return o, (torch.stack(states) if states else v.new_zeros(0, H, D, D))


def logprobs(logits, tokens, temperature=1.0):
    """(log probability of tokens, entropy) of finite or -inf logits, float64, differentiable."""
    x = logits / temperature
    lp = torch.log_softmax(x, -1)
    p = lp.exp()
    H = -torch.where(p > 0, p * torch.where(p > 0, lp, torch.zeros_like(lp)), torch.zeros_like(lp)).sum(-1)
    return lp.gather(1, tokens[:, None])[:, 0], H
