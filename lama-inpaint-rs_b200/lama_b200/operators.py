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
autograd.  Wrong arguments and GPU errors raise `LamaError`; a bounded wait of a kernel that ran out
is reported by `check_operators`.
"""

from __future__ import annotations

import ctypes
import threading
from dataclasses import dataclass, field
from struct import Struct
from typing import NamedTuple

import torch
from torch import Tensor

from .engine import LamaError, lib

__all__ = ["Checkpoint8", "check_operators", "checkpoint_restore", "checkpoint_store", "gated_residual_norm",
           "gated_residual_norm_backward", "linear_attention", "linear_attention_backward",
           "linear_attention_step"]

EINVAL = -1
GROUP = 128  # channels that share a scale of an 8-bit checkpoint
F32, I8, I32 = torch.float32, torch.int8, torch.int32
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}

# The header's structures, packed: a call of a small operator takes the host longer than the GPU, and
# ctypes.Structure objects cost several times a packed string.
_ROWS = "Pqqqi4x"                                     # lama_rows
_pack_rows = Struct("@" + _ROWS).pack
_pack_attention = Struct("@6i" + 3 * _ROWS + "3Pf4x").pack  # lama_attention
_pack_grads = Struct("@" + 4 * _ROWS + "2P").pack     # lama_attention_grads
_pack_norm = Struct("@i4xqi4xPqq3P2f").pack           # lama_norm
_pack_norm_grads = Struct("@4P4q12P").pack            # lama_norm_grads


class _Message(threading.local):
    def __init__(self):
        self.buf = ctypes.create_string_buffer(256)


_err = _Message()  # the library's message of this thread's last call
_current_stream = torch._C._cuda_getCurrentRawStream


def _refuse(msg):
    raise LamaError(EINVAL, msg)


def _check(rc):
    if rc < 0:
        raise LamaError(int(rc), _err.buf.value.decode())
    return rc


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _first(t, name, ndim=None):
    """A call's first tensor: on a CUDA device and of a supported type.  Returns the device's index."""
    if not isinstance(t, Tensor):
        _refuse(f"{name} is not a tensor")
    dev = t.get_device() if t.is_cuda else -1
    if dev < 0:
        _refuse(f"{name} is not on a CUDA device")
    if t.dtype not in _TYPES:
        _refuse(f"{name} has type {t.dtype}; float32, float16 and bfloat16 are supported")
    if ndim is not None and t.dim() != ndim:
        _refuse(f"{name} has {t.dim()} dimensions, not {ndim}")
    return dev


def _also(t, name, dev, dtype, shape=None):
    """Another tensor of the call: on the same device, of the given type and, unless None, shape."""
    if not isinstance(t, Tensor):
        _refuse(f"{name} is not a tensor")
    if not t.is_cuda or t.get_device() != dev:
        _refuse(f"{name} is on {t.device}, not on cuda:{dev}")
    if t.dtype is not dtype:
        _refuse(f"{name} has type {t.dtype}, not {dtype}")
    if shape is not None and t.shape != shape:
        _refuse(f"{name} has shape {tuple(t.shape)}, not {tuple(shape)}")


def check_operators(device=None) -> None:
    """Wait for the device and raise `LamaError` if a kernel's bounded wait ran out since the last call."""
    dev = torch.cuda.current_device() if device is None else torch.device(device).index or 0
    _check(lib().lama_operator_status(dev, _err.buf, 256))


# ------------------------------------------------------------------ linear attention

def _unit(t):
    """The tensor itself where the kernels take its strides at full speed, else a contiguous copy: rows have
    to be contiguous, and bfloat16 rows of a multiple of 8 channels on 16-byte boundaries (the copy then
    goes through the same kernel as a contiguous tensor, to the same bits)."""
    shape, stride = t.shape, t.stride()
    if stride[-1] != 1 and shape[-1] != 1:
        return t.contiguous()
    if t.dtype is torch.bfloat16 and shape[-1] % 8 == 0:
        if t.dim() == 4 and shape[1] > 1 and stride[1] == 0:
            return t.contiguous()
        if t.data_ptr() % 16 or any(s % 8 and n > 1 for n, s in zip(shape[:-1], stride)):
            return t.clone(memory_format=torch.contiguous_format)
    return t


def _rows(t):
    """[B,T,n,D] (or [B,n,D]) as the fields of a lama_rows."""
    n, s = t.shape, t.stride()  # a lone row's stride is arbitrary
    if t.dim() == 4:
        return (t.data_ptr(), s[0] if n[0] > 1 else 0, s[1] if n[1] > 1 else 0, s[2] if n[2] > 1 else 0, n[2])
    return t.data_ptr(), s[0] if n[0] > 1 else 0, 0, s[1] if n[1] > 1 else 0, n[1]


def _attention(q, k, v, log_decay, scale, initial_state, lengths, ndim):
    dev = _first(q, "q", ndim)
    dtype, shape = q.dtype, q.shape
    for t, name in ((k, "k"), (v, "v")):
        _also(t, name, dev, dtype)
        if t.dim() != ndim or t.shape[:-2] != shape[:-2]:
            _refuse(f"{name} has shape {tuple(t.shape)}, which does not go with q's {tuple(shape)}")
    dk, dv = shape[-1], v.shape[-1]
    if k.shape[-1] != dk:
        _refuse(f"q has {dk} channels a head and k {k.shape[-1]}")
    _also(log_decay, "log_decay", dev, F32)
    if log_decay.dim() != 1:
        _refuse(f"log_decay has {log_decay.dim()} dimensions, not 1")
    if log_decay.requires_grad and torch.is_grad_enabled():
        _refuse("log_decay has no gradient: the decays are constants of the layer")
    h = log_decay.shape[0]
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        n = t.shape[-2]
        if n < 1 or h % n or h < n:
            _refuse(f"{name} has {n} heads, which do not divide the {h} of log_decay")
    if not 1 <= dk <= 128 or not 1 <= dv <= 128:
        _refuse(f"head sizes {dk} and {dv} are not in 1..128")
    if initial_state is not None:
        _also(initial_state, "initial_state", dev, F32, (shape[0], h, dk, dv))
    if lengths is not None:
        _also(lengths, "lengths", dev, I32, (shape[0],))
    return dev, h, dk, dv, (dk ** -0.5 if scale is None else float(scale))


_needed = {}  # workspace bytes by sizes


def _workspace(args, key, backward, like):
    n = _needed.get((key, backward))
    if n is None:
        n = _check(lib().lama_linear_attention_workspace(args, backward, _err.buf, 256))
        if len(_needed) > 4096:
            _needed.clear()
        _needed[key, backward] = n
    return (like.new_empty(n, dtype=torch.uint8), n) if n else (None, 0)


def _attention_args(q, k, v, log_decay, scale, initial_state, lengths, h, dk, dv):
    code = _TYPES[q.dtype]
    b, t = q.shape[0], q.shape[1] if q.dim() == 4 else 1
    args = _pack_attention(code, b, t, h, dk, dv, *_rows(q), *_rows(k), *_rows(v), log_decay.data_ptr(),
                           _ptr(initial_state), _ptr(lengths), scale)
    return args, (code, b, t, h, dk, dv, q.shape[-2], k.shape[-2], v.shape[-2])


def _contiguous(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def _attention_forward(q, k, v, log_decay, scale, initial_state, lengths, return_state):
    dev, h, dk, dv, scale = _attention(q, k, v, log_decay, scale, initial_state, lengths, 4)
    q, k, v, log_decay = _unit(q), _unit(k), _unit(v), _contiguous(log_decay)
    b, t = q.shape[:2]
    o = q.new_empty((b, t, h, dv))
    state = q.new_empty((b, h, dk, dv), dtype=F32) if return_state else None
    if b == 0 or t == 0:
        if return_state:
            state.zero_() if initial_state is None else state.copy_(initial_state)
        return o, state
    initial_state, lengths = _contiguous(initial_state), _contiguous(lengths)
    args, key = _attention_args(q, k, v, log_decay, scale, initial_state, lengths, h, dk, dv)
    w, n = _workspace(args, key, 0, q)
    _check(lib().lama_linear_attention(args, _pack_rows(*_rows(o)), _ptr(state), _ptr(w), n, dev,
                                       _current_stream(dev), _err.buf, 256))
    return o, state


class _LinearAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, scale, initial_state, lengths):
        ctx.save_for_backward(q, k, v, log_decay, initial_state, lengths)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return _attention_forward(q, k, v, log_decay, scale, initial_state, lengths, True)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_o, grad_state):
        q, k, v, log_decay, initial_state, lengths = ctx.saved_tensors
        if grad_o is None:
            grad_o = q.new_zeros(*q.shape[:2], log_decay.numel(), v.shape[-1])
        dq, dk, dv, ds = linear_attention_backward(grad_o, q, k, v, log_decay, scale=ctx.scale,
                                                   initial_state=initial_state, lengths=lengths,
                                                   grad_state=grad_state)
        return dq, dk, dv, None, None, ds, None


def linear_attention(q, k, v, log_decay, *, scale=None, initial_state=None, lengths=None, return_state=False):
    """Linear attention with a decay for each head over whole sequences.

    S_t = exp(log_decay[h]) S_{t-1} + k_t v_t^T,  o_t = scale q_t S_t

    q, k: [B,T,n,dk], v: [B,T,n,dv], each with its own number n of heads that divides the H heads of
    log_decay [H] (float32, a constant of the layer; -inf is no memory): a head is shared by H/n
    neighbours.  Any strides.  scale: 1/sqrt(dk) unless given.  initial_state: [B,H,dk,dv] float32,
    zeros unless given.  lengths: [B] int32, the tokens of each sequence (later ones are not read, their
    outputs are 0).  Returns o [B,T,H,dv], or (o, state after the last token) with return_state.
    """
    grads = torch.is_grad_enabled() and any(isinstance(t, Tensor) and t.requires_grad
                                            for t in (q, k, v, initial_state))
    if grads:
        o, state = _LinearAttention.apply(q, k, v, log_decay, scale, initial_state, lengths)
    else:
        o, state = _attention_forward(q, k, v, log_decay, scale, initial_state, lengths, return_state)
    return (o, state) if return_state else o


def linear_attention_backward(grad_o, q, k, v, log_decay, *, scale=None, initial_state=None, lengths=None,
                              grad_state=None):
    """(dq, dk, dv, d_initial_state) of `linear_attention` for the gradients grad_o [B,T,H,dv] of its output
    and grad_state (None: zeros) of its final state; d_initial_state is None without an initial_state."""
    dev, h, dk, dv, scale = _attention(q, k, v, log_decay, scale, initial_state, lengths, 4)
    b, t = q.shape[:2]
    _also(grad_o, "grad_o", dev, q.dtype, (b, t, h, dv))
    if grad_state is not None:
        _also(grad_state, "grad_state", dev, F32, (b, h, dk, dv))
    q, k, v, grad_o, log_decay = _unit(q), _unit(k), _unit(v), _unit(grad_o), _contiguous(log_decay)
    grads = [x.new_empty(x.shape) for x in (q, k, v)]
    ds = None if initial_state is None else initial_state.new_empty(initial_state.shape)
    if b == 0 or t == 0:
        if ds is not None:
            ds.zero_() if grad_state is None else ds.copy_(grad_state)
        return (*grads, ds)
    initial_state, lengths, grad_state = _contiguous(initial_state), _contiguous(lengths), _contiguous(grad_state)
    args, key = _attention_args(q, k, v, log_decay, scale, initial_state, lengths, h, dk, dv)
    g = _pack_grads(*_rows(grad_o), *_rows(grads[0]), *_rows(grads[1]), *_rows(grads[2]), _ptr(grad_state), _ptr(ds))
    w, n = _workspace(args, key, 1, q)
    _check(lib().lama_linear_attention_backward(args, g, _ptr(w), n, dev, _current_stream(dev), _err.buf, 256))
    return (*grads, ds)


def linear_attention_step(q, k, v, log_decay, state, *, scale=None, slots=None, out_state=None):
    """One token of `linear_attention` for each row: S <- exp(log_decay) S + k v^T, o = scale q S.

    q, k: [B,n,dk], v: [B,n,dv] (heads shared as in `linear_attention`); state: [N,H,dk,dv] float32,
    contiguous, updated in place unless out_state, a separate buffer of its shape, takes the new states.
    slots: [B] int32, the state of each row, no slot twice (row b has slot b unless given); a slot
    outside 0..N-1 marks an unused row, whose output is 0.  Returns o [B,H,dv].  Has no gradient.
    """
    dev, h, dk, dv, scale = _attention(q, k, v, log_decay, scale, None, None, 3)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                    or isinstance(state, Tensor) and state.requires_grad):
        _refuse("a step has no gradient: call it under torch.no_grad() or use linear_attention")
    b = q.shape[0]
    _also(state, "state", dev, F32)
    shape = state.shape
    if len(shape) != 4 or shape[1:] != (h, dk, dv) or not state.is_contiguous():
        _refuse(f"state is not a contiguous tensor of shape (slots, {h}, {dk}, {dv})")
    if out_state is None:
        out_state = state
    else:
        _also(out_state, "out_state", dev, F32, shape)
        if not out_state.is_contiguous():
            _refuse("out_state is not contiguous")
    if slots is not None:
        _also(slots, "slots", dev, I32, (b,))
        slots = _contiguous(slots)
    elif shape[0] < b:
        _refuse(f"{shape[0]} states for {b} rows")
    q, k, v, log_decay = _last_unit(q), _last_unit(k), _last_unit(v), _contiguous(log_decay)
    o = q.new_empty((b, h, dv))
    if b == 0:
        return o
    if shape[0] == 0:
        return o.zero_()
    args, _ = _attention_args(q, k, v, log_decay, scale, None, None, h, dk, dv)
    _check(lib().lama_linear_attention_step(args, _pack_rows(*_rows(o)), state.data_ptr(), out_state.data_ptr(),
                                            shape[0], _ptr(slots), dev, _current_stream(dev), _err.buf, 256))
    return o


def _last_unit(t):
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


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


def _row_view(t):
    """[...,C] as a matrix of rows with one stride between them (a copy where its strides do not allow that)."""
    if t.dim() != 2:
        t = t.view(-1, t.shape[-1]) if t.is_contiguous() else t.flatten(0, -2) if t.dim() > 1 else t[None]
    n, s = t.shape, t.stride()
    if n[1] > 1 and s[1] != 1 or n[0] > 1 and s[0] < n[1]:
        t = t.contiguous()
    return t


def _row_stride(m):
    return m.stride(0) if m.shape[0] > 1 else m.shape[1]


def _empty_checkpoint(x):
    shape = x.shape
    return Checkpoint8(x.new_empty(shape, dtype=I8),
                       x.new_empty((*shape[:-1], (shape[-1] + GROUP - 1) // GROUP), dtype=F32), x.dtype)


def checkpoint_store(x) -> Checkpoint8:
    """x [...,C] in 8 bits, a scale for each row and group of 128 channels."""
    dev = _first(x, "x")
    if x.dim() < 1:
        _refuse("x has no channels")
    x = _plain(x)
    c = _empty_checkpoint(x)
    if x.numel():
        m = _row_view(x)
        _check(lib().lama_checkpoint_store(m.data_ptr(), _TYPES[x.dtype], m.shape[0], m.shape[1], _row_stride(m),
                                           c.codes.data_ptr(), c.scales.data_ptr(), dev, _current_stream(dev),
                                           _err.buf, 256))
    return c


def _plain(t):
    """Without autograd's view of it."""
    return t.detach() if t is not None and t.requires_grad else t


def checkpoint_restore(ckpt: Checkpoint8, dtype=None) -> torch.Tensor:
    """The activation a checkpoint stands for, in its own type unless `dtype` is given."""
    if not isinstance(ckpt, Checkpoint8):
        _refuse("not a Checkpoint8")
    dtype = ckpt.dtype if dtype is None else dtype
    if dtype not in _TYPES:
        _refuse(f"type {dtype} is not supported")
    codes, scales = ckpt.codes, ckpt.scales
    if not isinstance(codes, Tensor) or not codes.is_cuda or codes.dtype is not I8 or codes.dim() < 1:
        _refuse("codes is not an int8 tensor on a CUDA device")
    dev, shape = codes.get_device(), codes.shape
    _also(scales, "scales", dev, F32, (*shape[:-1], (shape[-1] + GROUP - 1) // GROUP))
    x = codes.new_empty(shape, dtype=dtype)
    if x.numel():
        codes, scales, c = _contiguous(codes), _contiguous(scales), shape[-1]
        _check(lib().lama_checkpoint_restore(codes.data_ptr(), scales.data_ptr(), _TYPES[dtype], x.numel() // c, c, c,
                                             x.data_ptr(), dev, _current_stream(dev), _err.buf, 256))
    return x


# ------------------------------------------------------------------ norms, gate and residual

@dataclass
class SavedNorm:
    """What `gated_residual_norm` keeps for its backward pass."""
    args: tuple = field(repr=False)  # post_weight, pre_weight, gate (as given), residual_scale, eps
    y: torch.Tensor | Checkpoint8
    u: torch.Tensor | Checkpoint8 | None
    post_rstd: torch.Tensor | None
    pre_rstd: torch.Tensor | None
    shape: tuple
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


def _gate_rows(gate, shape):
    """A gate that broadcasts over x's shape as (its rows as a matrix, rows of x that share one of them).
    Its dimensions of size 1 have to be the innermost of x's row dimensions."""
    lead = shape[:-1]
    g = [1] * (len(lead) - (gate.dim() - 1)) + list(gate.shape[:-1])
    if gate.dim() < 1 or gate.dim() > len(shape) or gate.shape[-1] != shape[-1]:
        _refuse(f"a gate of shape {tuple(gate.shape)} does not broadcast over {tuple(shape)}")
    per, whole = 1, False
    for n, m in zip(reversed(g), reversed(lead)):
        if n == m and (m != 1 or whole):
            whole = True
        elif n == 1 and not whole:
            per *= m
        elif n != m:
            _refuse(f"a gate of shape {tuple(gate.shape)} does not broadcast over {tuple(shape)} one gate row to "
                    "neighbouring rows; expand it")
    return _row_view(gate), per


def _vector(w, name, dev, c):
    """A weight [C] as contiguous float32."""
    if not isinstance(w, Tensor) or not w.is_cuda or w.get_device() != dev or w.dtype not in _TYPES or w.shape != (c,):
        _refuse(f"{name} is not a tensor of {c} channels on cuda:{dev}")
    w = _plain(w)
    return _contiguous(w if w.dtype is F32 else w.float())


def _norm_args(x, dev, post_weight, pre_weight, gate, residual_scale, eps):
    shape = x.shape
    c = shape[-1]
    scales = None
    if isinstance(residual_scale, Tensor):
        scales, residual_scale = _vector(residual_scale, "residual_scale", dev, c), 0.0
    if post_weight is not None:
        post_weight = _vector(post_weight, "post_weight", dev, c)
    if pre_weight is not None:
        pre_weight = _vector(pre_weight, "pre_weight", dev, c)
    rows, per, stride = None, 1, 0
    if gate is not None:
        _also(gate, "gate", dev, x.dtype)
        rows, per = _gate_rows(_plain(gate), shape)
        stride = _row_stride(rows)
    a = _pack_norm(_TYPES[x.dtype], x.numel() // c, c, _ptr(rows), per, stride, _ptr(post_weight), _ptr(pre_weight),
                   _ptr(scales), float(residual_scale), float(eps))
    return a, (post_weight, pre_weight, rows, scales)  # the tensors a points to


def _norm_forward(x, y, post_weight, pre_weight, gate, residual_scale, eps, save):
    dev = _first(x, "x")
    shape = x.shape
    if len(shape) < 1 or shape[-1] < 1:
        _refuse("x has no channels")
    _also(y, "y", dev, x.dtype, shape)
    if save not in (None, "full", "int8"):
        _refuse(f"save is {save!r}, not None, 'full' or 'int8'")
    if not float(eps) >= 0:
        _refuse("eps must not be negative")
    x, y = _plain(x), _plain(y)
    u = x.new_empty(shape)
    n = None if pre_weight is None else x.new_empty(shape)
    ry = ru = cy = cu = None
    if save:
        ry = None if post_weight is None else x.new_empty(shape[:-1], dtype=F32)
        ru = None if pre_weight is None else x.new_empty(shape[:-1], dtype=F32)
        if save == "int8":
            cy = _empty_checkpoint(y)
            cu = None if pre_weight is None else _empty_checkpoint(u)
    if x.numel():
        a, keep = _norm_args(x, dev, post_weight, pre_weight, gate, residual_scale, eps)
        mx, my = _row_view(x), _row_view(y)
        _check(lib().lama_gated_residual_norm(
            a, mx.data_ptr(), _row_stride(mx), my.data_ptr(), _row_stride(my), u.data_ptr(), _ptr(n), _ptr(ry), _ptr(ru),
            cy and cy.codes.data_ptr(), cy and cy.scales.data_ptr(), cu and cu.codes.data_ptr(),
            cu and cu.scales.data_ptr(), dev, _current_stream(dev), _err.buf, 256))
    saved = None
    if save:
        saved = SavedNorm((post_weight, pre_weight, gate, residual_scale, eps), cy if cy is not None else y,
                          None if pre_weight is None else cu if cu is not None else u, ry, ru, shape, x.dtype)
    return u, n, saved


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
        ctx.shape, ctx.dtype = x.shape, x.dtype
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
                          ctx.shape, ctx.dtype)
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
    if torch.is_grad_enabled() and any(isinstance(t, Tensor) and t.requires_grad for t in ts):
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
    int8 = isinstance(y, Checkpoint8)
    some = y.codes if int8 else y
    shape, dtype, dev = saved.shape, saved.dtype, some.get_device()
    c = shape[-1]
    if grad_u is not None:
        _also(grad_u, "grad_u", dev, dtype, shape)
    if grad_n is not None:
        _also(grad_n, "grad_n", dev, dtype, shape)

    def vector(w):
        return some.new_empty(c, dtype=F32) if isinstance(w, Tensor) else None

    dx, dy = some.new_empty(shape, dtype=dtype), some.new_empty(shape, dtype=dtype)
    dpost, dpre, dscale = vector(post_weight), vector(pre_weight), vector(residual_scale)
    dgate = None if gate is None else some.new_empty(gate.shape, dtype=dtype)
    if dx.numel():
        a, keep = _norm_args(dx, dev, post_weight, pre_weight, gate, residual_scale, eps)
        mu = None if grad_u is None else _row_view(_plain(grad_u))
        mn = None if grad_n is None else _row_view(_plain(grad_n))
        my = mz = None
        if not int8:
            my, mz = _row_view(y), None if u is None else _row_view(u)
        has_u = int8 and u is not None
        g = _pack_norm_grads(_ptr(mu), _ptr(mn), _ptr(my), _ptr(mz), *(0 if m is None else _row_stride(m)
                                                                      for m in (mu, mn, my, mz)),
                             y.codes.data_ptr() if int8 else 0, u.codes.data_ptr() if has_u else 0,
                             y.scales.data_ptr() if int8 else 0, u.scales.data_ptr() if has_u else 0,
                             _ptr(saved.post_rstd), _ptr(saved.pre_rstd), dx.data_ptr(), dy.data_ptr(), _ptr(dgate),
                             _ptr(dpost), _ptr(dpre), _ptr(dscale))
        n = _check(lib().lama_gated_residual_norm_workspace(a, _err.buf, 256))
        w = some.new_empty(n, dtype=torch.uint8)
        _check(lib().lama_gated_residual_norm_backward(a, g, w.data_ptr(), n, dev, _current_stream(dev), _err.buf, 256))
    else:
        for t in (dgate, dpost, dpre, dscale):
            if t is not None:
                t.zero_()

    def like(g, w):
        return g if g is None or w.dtype is F32 else g.to(w.dtype)

    return NormGradients(dx, dy, like(dpost, post_weight), like(dpre, pre_weight), dgate, like(dscale, residual_scale))
