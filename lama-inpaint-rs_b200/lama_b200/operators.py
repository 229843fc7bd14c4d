"""Token-mixer operators on CUDA tensors (include/lama_b200.h, no counterpart in the reference).

Three operators for a block that mixes the tokens of a latent plane (or of any sequence), in
inference and training:

* `linear_attention`, `linear_attention_backward`, `linear_attention_step`: linear attention with a
  decay for each head, over whole sequences and one token at a time;
* `gated_residual_norm`, `gated_residual_norm_backward`: the norm after a block, its gate and
  residual scale, the residual sum and the norm before the next block in one pass;
* `checkpoint_store`, `checkpoint_restore`: an activation kept in 8 bits for the backward pass, which
  `gated_residual_norm(save="int8")` also writes and its backward pass reads.

Tensors are torch tensors on one CUDA device, of type float32, float16 or bfloat16; work is queued on
torch's current stream of that device.  `linear_attention` and `gated_residual_norm` take part in
autograd (backward mode, once; tensors with forward-mode tangents are refused).  Wrong arguments and
GPU errors raise `LamaError`; a bounded wait of a kernel that ran out is reported by
`check_operators`.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass, field
from typing import NamedTuple

import torch
from torch import Tensor

from . import _operators as _native  # csrc/torch_binding.cpp: argument checks, outputs, the library's calls
from .engine import LamaError, lib

__all__ = ["Checkpoint8", "check_operators", "checkpoint_restore", "checkpoint_store", "gated_residual_norm",
           "gated_residual_norm_backward", "linear_attention", "linear_attention_backward",
           "linear_attention_step"]

EINVAL = -1
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_grad_enabled = torch.is_grad_enabled

_native.setup(LamaError, *(ctypes.cast(getattr(lib(), "lama_" + n), ctypes.c_void_p).value for n in (
    "linear_attention_workspace", "linear_attention", "linear_attention_backward", "linear_attention_step",
    "gated_residual_norm", "gated_residual_norm_workspace", "gated_residual_norm_backward", "checkpoint_store",
    "checkpoint_restore")))


def _refuse(msg):
    raise LamaError(EINVAL, msg)


def _learns(*ts):
    return any(isinstance(t, Tensor) and t.requires_grad for t in ts)


def check_operators(device=None) -> None:
    """Wait for the device and raise `LamaError` if a kernel's bounded wait ran out since the last call."""
    dev = torch.device("cuda" if device is None else device)
    if dev.type != "cuda":
        _refuse(f"{dev} is not a CUDA device")
    dev = torch.cuda.current_device() if dev.index is None else dev.index
    err = ctypes.create_string_buffer(256)
    rc = lib().lama_operator_status(dev, err, 256)
    if rc < 0:
        raise LamaError(rc, err.value.decode())


# ------------------------------------------------------------------ linear attention

class _LinearAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, scale, initial_state, lengths, return_state):
        ctx.save_for_backward(q, k, v, log_decay, initial_state, lengths)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        o, state = _native.attention(q, k, v, log_decay, scale, initial_state, lengths, return_state)
        return (o, state) if return_state else o

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_o, grad_state=None):
        q, k, v, log_decay, initial_state, lengths = ctx.saved_tensors
        if grad_o is None:
            grad_o = q.new_zeros(*q.shape[:2], log_decay.numel(), v.shape[-1])
        dq, dk, dv, ds = linear_attention_backward(grad_o, q, k, v, log_decay, scale=ctx.scale,
                                                   initial_state=initial_state, lengths=lengths,
                                                   grad_state=grad_state)
        return dq, dk, dv, None, None, ds, None, None


def linear_attention(q, k, v, log_decay, *, scale=None, initial_state=None, lengths=None, return_state=False):
    """Linear attention with a decay for each head over whole sequences.

    S_t = exp(log_decay[h]) S_{t-1} + k_t v_t^T,  o_t = scale q_t S_t

    q, k: [B,T,n,dk], v: [B,T,n,dv], each with its own number n of heads that divides the H heads of
    log_decay [H] (float32, a constant of the layer; -inf is no memory): a head is shared by H/n
    neighbours.  Any strides.  scale: 1/sqrt(dk) unless given.  initial_state: [B,H,dk,dv] float32,
    zeros unless given.  lengths: [B] int32, the tokens of each sequence (later ones are not read, their
    outputs are 0).  Returns o [B,T,H,dv], or (o, state after the last token) with return_state.
    """
    if _grad_enabled() and _learns(q, k, v, initial_state):
        if _learns(log_decay):  # inside the function gradients are off, and the binding's own check with them
            _refuse("log_decay has no gradient: the decays are constants of the layer")
        return _LinearAttention.apply(q, k, v, log_decay, scale, initial_state, lengths, bool(return_state))
    o, state = _native.attention(q, k, v, log_decay, scale, initial_state, lengths, bool(return_state))
    return (o, state) if return_state else o


def linear_attention_backward(grad_o, q, k, v, log_decay, *, scale=None, initial_state=None, lengths=None,
                              grad_state=None):
    """(dq, dk, dv, d_initial_state) of `linear_attention` for the gradients grad_o [B,T,H,dv] of its output
    and grad_state (None: zeros) of its final state; d_initial_state is None without an initial_state."""
    return _native.attention_backward(grad_o, q, k, v, log_decay, scale, initial_state, lengths, grad_state)


def linear_attention_step(q, k, v, log_decay, state, *, scale=None, slots=None, out_state=None):
    """One token of `linear_attention` for each row: S <- exp(log_decay) S + k v^T, o = scale q S.

    q, k: [B,n,dk], v: [B,n,dv] (heads shared as in `linear_attention`); state: [N,H,dk,dv] float32,
    contiguous, updated in place unless out_state, a separate buffer of its shape, takes the new states.
    slots: [B] int32, the state of each row, no slot twice (row b has slot b unless given); a slot
    outside 0..N-1 marks an unused row, whose output is 0.  Returns o [B,H,dv].  Has no gradient.
    """
    return _native.attention_step(q, k, v, log_decay, state, scale, slots, out_state)


# ------------------------------------------------------------------ 8-bit checkpoints

@dataclass
class Checkpoint8:
    """An activation in 8 bits: codes [...,C] int8, scales [...,ceil(C/128)] float32, the type it had."""
    codes: torch.Tensor
    scales: torch.Tensor
    dtype: torch.dtype

    @property
    def nbytes(self) -> int:
        return self.codes.nbytes + self.scales.nbytes


def checkpoint_store(x) -> Checkpoint8:
    """x [...,C] in 8 bits, a scale for each row and group of 128 channels.  Has no gradient."""
    codes, scales = _native.store(x)
    return Checkpoint8(codes, scales, x.dtype)


def checkpoint_restore(ckpt: Checkpoint8, dtype=None) -> torch.Tensor:
    """The activation a checkpoint stands for, in its own type unless `dtype` is given."""
    if not isinstance(ckpt, Checkpoint8):
        _refuse("not a Checkpoint8")
    dtype = ckpt.dtype if dtype is None else dtype
    if dtype not in _TYPES:
        _refuse(f"type {dtype} is not supported")
    return _native.restore(ckpt.codes, ckpt.scales, _TYPES[dtype])


# ------------------------------------------------------------------ norms, gate and residual

@dataclass
class SavedNorm:
    """What `gated_residual_norm` keeps for its backward pass."""
    args: tuple = field(repr=False)  # post_weight, pre_weight, gate (as given), residual_scale, eps
    y: torch.Tensor | Checkpoint8
    u: torch.Tensor | Checkpoint8 | None
    post_rstd: torch.Tensor | None
    pre_rstd: torch.Tensor | None
    dtype: torch.dtype

    @property
    def nbytes(self) -> int:
        return sum(t.nbytes for t in (self.y, self.u, self.post_rstd, self.pre_rstd) if t is not None)


class NormGradients(NamedTuple):
    x: torch.Tensor
    y: torch.Tensor
    post_weight: torch.Tensor | None
    pre_weight: torch.Tensor | None
    gate: torch.Tensor | None
    residual_scale: torch.Tensor | None


_SAVES = {None: 0, "full": 1, "int8": 2}


def _norm_forward(x, y, post_weight, pre_weight, gate, residual_scale, eps, save):
    if save not in _SAVES:
        _refuse(f"save is {save!r}, not None, 'full' or 'int8'")
    u, n, ry, ru, cy, sy, cu, su = _native.norm(x, y, post_weight, pre_weight, gate, residual_scale, eps, _SAVES[save])
    if not save:
        return u, n, None
    if save == "int8":
        ky, ku = Checkpoint8(cy, sy, x.dtype), None if cu is None else Checkpoint8(cu, su, x.dtype)
    else:
        ky, ku = y.detach(), None if n is None else u
    return u, n, SavedNorm((post_weight, pre_weight, gate, residual_scale, eps), ky, ku, ry, ru, x.dtype)


class _GatedResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, post_weight, pre_weight, gate, residual_scale, eps, int8):
        u, n, saved = _norm_forward(x, y, post_weight, pre_weight, gate, residual_scale, eps,
                                    "int8" if int8 else "full")
        # everything goes through save_for_backward, so that autograd sees in-place changes and frees it in time
        flat = []
        for t in (saved.y, saved.u):
            flat += [t.codes, t.scales] if isinstance(t, Checkpoint8) else [t, None]
        scale = residual_scale if isinstance(residual_scale, Tensor) else None
        ctx.save_for_backward(*flat, saved.post_rstd, saved.pre_rstd, post_weight, pre_weight, gate, scale)
        ctx.int8, ctx.scale, ctx.eps = int8, None if scale is not None else residual_scale, eps
        ctx.dtype = x.dtype
        ctx.set_materialize_grads(False)
        return (u, n) if n is not None else u

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_u, grad_n=None):
        y, ys, u, us, ry, ru, post_weight, pre_weight, gate, scale = ctx.saved_tensors
        if ctx.int8:
            y = Checkpoint8(y, ys, ctx.dtype)
            u = None if u is None else Checkpoint8(u, us, ctx.dtype)
        saved = SavedNorm((post_weight, pre_weight, gate, ctx.scale if scale is None else scale, ctx.eps), y, u, ry, ru,
                          ctx.dtype)
        g = gated_residual_norm_backward(grad_u, grad_n, saved)
        return g.x, g.y, g.post_weight, g.pre_weight, g.gate, g.residual_scale, None, None


def gated_residual_norm(x, y, *, post_weight=None, pre_weight=None, gate=None, residual_scale=1.0, eps=1e-6, save=None):
    """The norm after a block, its gate and residual scale, the residual sum and the next block's norm.

    p = post_weight * rms_norm(y)   (p = y without post_weight)
    u = x + residual_scale * gate * p
    n = pre_weight * rms_norm(u)    (n = None without pre_weight)

    x, y: [...,C]; weights [C]; gate: None, or a tensor of x's type that broadcasts over x with its
    size-1 dimensions innermost ([B,1,C], [B,T,C], [C]); residual_scale: a number or [C].  Returns (u, n), or
    (u, n, saved) with save="full" (y and u themselves are kept) or save="int8" (8-bit checkpoints of
    them, written in the same pass): `gated_residual_norm_backward` takes `saved`.  Under autograd, "int8"
    keeps the checkpoints in the graph and `saved` is None.
    """
    ts = (x, y, post_weight, pre_weight, gate, residual_scale)
    if _grad_enabled() and _learns(*ts):
        if save not in (None, "full", "int8"):
            _refuse(f"save is {save!r}, not None, 'full' or 'int8'")
        out = _GatedResidualNorm.apply(*ts, eps, save == "int8")
        u, n = out if isinstance(out, tuple) else (out, None)
        return (u, n, None) if save else (u, n)
    u, n, saved = _norm_forward(*ts, eps, save)
    return (u, n, saved) if save else (u, n)


def gated_residual_norm_backward(grad_u, grad_n, saved) -> NormGradients:
    """Gradients of `gated_residual_norm` for those of u and n (either may be None: zeros)."""
    post_weight, pre_weight, gate, residual_scale, eps = saved.args
    y, u = saved.y, saved.u
    if isinstance(y, Checkpoint8):
        kept = y.codes, y.codes, y.scales, None if u is None else u.codes, None if u is None else u.scales
    else:
        kept = y, y, None, u, None
    dx, dy, dpost, dpre, dgate, dscale = _native.norm_backward(
        kept[0], _TYPES[saved.dtype], grad_u, grad_n, post_weight, pre_weight, gate, residual_scale, eps, *kept[1:],
        saved.post_rstd, saved.pre_rstd)

    def like(g, w):
        return g if g is None or w.dtype is torch.float32 else g.to(w.dtype)

    return NormGradients(dx, dy, like(dpost, post_weight), like(dpre, pre_weight), dgate, like(dscale, residual_scale))
