"""The gated delta rule on sm_100a: chunked over sequences, and token by token.

Per (sequence, value head), with S the fp32 ``[D, D]`` state (rows = key
channels), g the log decay and beta the write strength of a token:

    S' = exp(g_t) S_{t-1}          u_t = beta_t (v_t - S'^T k_t)
    S_t = S' + k_t u_t^T           o_t = scale * S_t^T q_t

Unlike ``kda_chunk``'s state, which only adds ``k^T v``, the rule first takes
out what the state already predicts for ``k_t``.  ``gated_delta_chunk`` runs it
over whole sequences (training, prefill) and ``gated_delta_step`` continues it
one token a call on a pool of states (serving); both hold the state in fp32 and
agree on it to a few parts in 1e6 (bf16 keys that repeat, at beta 1.9: 1e-4).

``kda_b200::delta_fwd / delta_bwd / delta_step`` are defined and implemented in
C++, autograd included (``csrc/torch_ops.cpp``), over the C ABI (``include/kda_sm100.h``): they run
on torch's current stream with workspace from the caching allocator, and can be
captured in CUDA graphs.  There is no CPU path.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import ops as _ops  # noqa: F401  (loads the library that defines the kda_b200 ops)

Tensor = torch.Tensor

_HALF = (torch.bfloat16, torch.float16)
_GATE = (torch.float32, torch.bfloat16, torch.float16)


def _empty_in_order_of(like: Tensor) -> Tensor:
    """The ops' rule for their [B, H, T, D] outputs: the input's strides where they are dense,
    [B, T, H, D] memory where it is time-major, else contiguous."""
    step, dense = 1, True
    for i in sorted((i for i in range(4) if like.shape[i] != 1), key=like.stride):
        dense = dense and like.stride(i) == step
        step = step * like.shape[i]
    if dense:
        return torch.empty_like(like)
    if like.stride(1) < like.stride(2):
        return like.new_empty(like.shape[0], like.shape[2], like.shape[1], like.shape[3]).transpose(1, 2)
    return like.new_empty(like.shape)


@torch.library.register_fake("kda_b200::delta_fwd")
def _(q, k, v, g, beta, scale, s0, cu_seqlens, want_state):
    n = v.shape[0] if cu_seqlens is None else cu_seqlens.shape[0] - 1
    D = v.shape[3]
    shape = (n, v.shape[1], D, D) if want_state else (0,)
    return _empty_in_order_of(v), q.new_empty(shape, dtype=torch.float32)


@torch.library.register_fake("kda_b200::delta_bwd")
def _(q, k, v, g, beta, scale, s0, cu_seqlens, dout, ds_T, need_ds0):
    n = v.shape[0] if cu_seqlens is None else cu_seqlens.shape[0] - 1
    D = v.shape[3]
    ds0 = q.new_empty((n, v.shape[1], D, D) if need_ds0 else (0,), dtype=torch.float32)
    return (_empty_in_order_of(q), _empty_in_order_of(k), _empty_in_order_of(v),
            g.new_empty(g.shape), beta.new_empty(beta.shape), ds0)


@torch.library.register_fake("kda_b200::delta_step")
def _(q, k, v, g, beta, state, state_indices, scale):
    return v.new_empty(v.shape)


def _validate(q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, names: str):
    dims = 4 if names == "chunk" else 3
    kind = "[B, H, T, D]" if dims == 4 else "[N, H, D]"
    if q.dim() != dims or v.dim() != dims:
        raise ValueError(f"q and v must be {kind}, got shapes {tuple(q.shape)} and {tuple(v.shape)}")
    if k.shape != q.shape:
        raise ValueError(f"k shape {tuple(k.shape)} != q shape {tuple(q.shape)}")
    if q.shape[0] != v.shape[0] or q.shape[2:] != v.shape[2:]:
        raise ValueError(f"q shape {tuple(q.shape)} and v shape {tuple(v.shape)} may differ in their heads only")
    H, Hk = v.shape[1], q.shape[1]
    if H and (not Hk or H % Hk):
        raise ValueError(f"{H} value heads cannot share {Hk} query/key heads evenly")
    if v.shape[-1] not in (64, 128):
        raise ValueError(f"the head dim must be 64 or 128, got {v.shape[-1]}")
    if q.dtype not in _HALF:
        raise TypeError(f"the delta rule takes bf16/fp16 q, k, v, got {q.dtype}")
    for n, t in (("k", k), ("v", v)):
        if t.dtype != q.dtype or t.device != q.device:
            raise TypeError(f"{n} must match q's dtype and device")
    for n, t in (("g", g), ("beta", beta)):
        if t.shape != v.shape[:-1]:
            raise ValueError(f"{n} must be {kind[:-4]}] = {tuple(v.shape[:-1])}, got {tuple(t.shape)}")
        if t.dtype not in _GATE or t.device != q.device:
            raise TypeError(f"{n} must be float32, bfloat16 or float16 on q's device")


def _need_cuda(q: Tensor):
    if q.device.type != "cuda":
        raise RuntimeError("the KDA sm_100a kernels need CUDA tensors (there is no CPU path)")


def _indices(t: Tensor, name: str, device: torch.device):
    if t.dim() != 1 or t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name} must be a one-dimensional int32 or int64 tensor")
    if t.device != device:
        raise TypeError(f"{name} must be on q's device")


def _check_chunk(q, k, v, g, beta, initial_state, cu_seqlens):
    _validate(q, k, v, g, beta, "chunk")
    B, H, T, D = v.shape
    n = B
    if cu_seqlens is not None:
        _indices(cu_seqlens, "cu_seqlens", q.device)
        if B != 1:
            raise ValueError(f"cu_seqlens packs sequences into one row: the batch must be 1, got {B}")
        if cu_seqlens.shape[0] < 1:
            raise ValueError("cu_seqlens needs at least one offset")
        if T > 1 << 24:
            raise ValueError(f"a packed row holds at most 2^24 tokens, got {T}")
        n = cu_seqlens.shape[0] - 1
    if initial_state is not None:
        if initial_state.shape != (n, H, D, D):
            raise ValueError(f"initial_state must be [sequences, H, D, D] = {(n, H, D, D)}, got {tuple(initial_state.shape)}")
        if initial_state.dtype != torch.float32 or initial_state.device != q.device:
            raise TypeError("initial_state must be float32 on q's device")
    _need_cuda(q)


def gated_delta_chunk(q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, *, scale: Optional[float] = None,
                      initial_state: Optional[Tensor] = None, cu_seqlens: Optional[Tensor] = None,
                      output_final_state: bool = True) -> Tuple[Tensor, Optional[Tensor]]:
    """The gated delta rule over sequences: returns ``(o, final_state)``.

    q, k: ``[B, Hk, T, D]``, v: ``[B, H, T, D]``, bf16/fp16 CUDA tensors of any
    strides (the ``[B, T, H, D]``-memory views of a layer's projections are used
    in place), D 64 or 128.  H is a multiple of Hk: value head h reads query/key
    head ``h // (H // Hk)``.  g, beta: ``[B, H, T]`` float32, bf16 or fp16; g is
    the log of the decay (at most 0 in use; below -110 it counts as -110, where
    the decay is 0 in fp32 already).  ``scale`` defaults to ``D ** -0.5``.

    ``cu_seqlens`` (int32 or int64, ``[n + 1]``, on the device, with B == 1) packs
    n sequences into the row (of at most 2^24 tokens): sequence i is tokens ``cu_seqlens[i]`` to
    ``cu_seqlens[i + 1]`` and starts from ``initial_state[i]``.  Sequences may be
    empty; tokens outside all of them get zero outputs and zero gradients.
    Offsets out of order or range are clamped and set a bit of
    ``device_status()``.  ``initial_state``: float32 ``[n or B, H, D, D]`` or None
    (zeros); ``final_state`` has that shape.

    Differentiable (once) in q, k, v, g, beta and initial_state, through o and
    final_state; gradients of shared heads are summed in a fixed order.  A NaN or
    infinity in a token reaches its own 64-token chunk and what follows in its
    sequence (earlier tokens of the chunk too), and no other sequence.

    States and gradients are fp32 whatever the inputs' type, of any size: in fp16 what a chunk
    computes is carried relative to the largest state, value and gradient of that chunk and head, with
    room for 2^9 times as much inside the chunk (a rule with ``beta |k|^2 <= 2`` stays far below);
    what is 2^12 times smaller than that keeps its bits, what is smaller still loses them one by one.
    """
    D = v.shape[-1] if v.dim() else 0
    try:
        o, s = torch.ops.kda_b200.delta_fwd(q, k, v, g, beta, float(D or 1) ** -0.5 if scale is None else float(scale),
                                            initial_state, cu_seqlens, bool(output_final_state))
    except RuntimeError:  # the op checks its arguments; say what is wrong with them
        _check_chunk(q, k, v, g, beta, initial_state, cu_seqlens)
        raise
    return o, (s if output_final_state else None)


def _check_step(q, k, v, g, beta, state, state_indices):
    _validate(q, k, v, g, beta, "step")
    N, H, D = v.shape
    if state.dim() != 4 or state.shape[1:] != (H, D, D):
        raise ValueError(f"state must be [states, H, D, D] with H, D = {H}, {D}, got {tuple(state.shape)}")
    if state.dtype != torch.float32 or state.device != q.device:
        raise TypeError("state must be float32 on q's device")
    if state_indices is not None:
        _indices(state_indices, "state_indices", q.device)
        if state_indices.shape[0] != N:
            raise ValueError(f"state_indices must be [N] = [{N}], got {tuple(state_indices.shape)}")
    elif N > state.shape[0]:
        raise ValueError(f"{N} rows need {N} states, got {state.shape[0]}")
    _need_cuda(q)


def gated_delta_step(q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, state: Tensor, *,
                     state_indices: Optional[Tensor] = None, scale: Optional[float] = None) -> Tensor:
    """One new token a row, on states updated in place: returns o ``[N, H, D]``.

    q, k: ``[N, Hk, D]``, v: ``[N, H, D]`` bf16/fp16; g, beta: ``[N, H]``;
    ``state``: float32 ``[states, H, D, D]``, e.g. the ``final_state`` of
    ``gated_delta_chunk``; it may be a strided view of a larger pool as long as
    each ``[D, D]`` is contiguous.  Row n uses state ``state_indices[n]`` (int32 or
    int64), or state n without them.  A negative index marks a padded row: its o
    is zero and no state changes.  An index past the pool does the same and sets a
    bit of ``device_status()``.  Rows that name the same state are applied in row
    order (looking for them takes 4% of a call of 256 rows, 74% more at 8192).  The step has no gradient: differentiate ``gated_delta_chunk``.
    """
    D = v.shape[-1] if v.dim() else 0
    try:
        return torch.ops.kda_b200.delta_step(q, k, v, g, beta, state, state_indices,
                                             float(D or 1) ** -0.5 if scale is None else float(scale))
    except NotImplementedError:  # gradients asked for, or tensors on the CPU
        if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, g, beta, state)):
            raise
        _check_step(q, k, v, g, beta, state, state_indices)
        raise
    except RuntimeError:
        _check_step(q, k, v, g, beta, state, state_indices)
        raise
