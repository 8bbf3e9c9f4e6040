"""Gated linear recurrence: the LSTM cell without its recurrent product.

    c_t = sigmoid(f_t) c_{t-1} + sigmoid(i_t) tanh(n_t)
    h_t = sigmoid(o_t) tanh(c_t)

``gates`` is [T, B, 4H], the pre-activations in the framework's gate order
(i, f, o, n): one GEMM over the whole window makes them, since no gate reads
``h_{t-1}``. Time is then a scan, not a chain of T products.

Types and layouts
  * ``gates``, ``h`` and their gradients: float32, bfloat16 or float16. The
    last axis is dense; time and batch may have any strides (batch-first
    storage is ``x.transpose(0, 1)``). ``h`` and ``dgates`` are stored in the
    order of ``gates``.
  * states (``c0``, ``cT`` and their gradients): float32 [B, H], finite.
    ``None`` stands for zeros. A NaN stays in its channel, from its step on.
  * ``lengths``: int32 or int64 [B] on the same device, values outside
    [0, T] count as the nearer end. From ``lengths[b]`` on row b keeps its
    state, its ``h`` and ``dgates`` are zero, and what stands in ``gates``
    and ``dh`` there has no effect, NaN included.

On the GPU every function runs the HIP kernels on the current stream of the
tensors' device; on the CPU (or with ZAREMBA_AMD_FORCE_EAGER=1) it runs the
eager math of ops/functional.py. All of them may be captured in a HIP graph;
a captured training step calls glr_forward and glr_backward themselves, which
need no autograd. Windows of up to 128 steps are one launch; longer ones two,
with a workspace of 8 bytes for each channel and 128 steps (64 backward, and
forward from 16384 channels on). Their blocks wait for each other, a bounded
time: should one ever give up, the states from its steps on are NaN.
"""

from __future__ import annotations

import torch

from .. import _C
from . import functional as F_ref


def _eager(gates: torch.Tensor) -> bool:
    return not gates.is_cuda or _C.force_eager_env()


def _check_eager(op, gates, dims, **states):
    if gates.dim() != dims or gates.size(-1) % 4:
        raise RuntimeError(f"{op}: gates must be "
                           f"{'[T, B, 4H]' if dims == 3 else '[B, 4H]'}, "
                           f"got {list(gates.shape)}")
    if not gates.is_floating_point():
        raise RuntimeError(f"{op}: gates must be float32, float16 or "
                           f"bfloat16, got {gates.dtype}")
    want = (gates.size(-2), gates.size(-1) // 4)
    for name, c in states.items():
        if c is None:
            continue
        if c.dtype not in (torch.float32, torch.float64):
            raise RuntimeError(f"{op}: {name} must be float32, got {c.dtype}")
        if tuple(c.shape) != want:
            raise RuntimeError(f"{op}: {name} must be {list(want)}, got "
                               f"{list(c.shape)}")


def _check_lengths(op, gates, lengths):
    if lengths is None:
        return
    if lengths.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f"{op}: lengths must be int32 or int64, got "
                           f"{lengths.dtype}")
    if tuple(lengths.shape) != (gates.size(1),):
        raise RuntimeError(f"{op}: lengths must be [{gates.size(1)}], got "
                           f"{list(lengths.shape)}")


def _check_like_h(op, name, x, gates, width):
    if x is None:
        return
    want = (gates.size(0), gates.size(1), width)
    if tuple(x.shape) != want or x.dtype != gates.dtype:
        raise RuntimeError(f"{op}: {name} must be {list(want)} of the gates' "
                           f"type {gates.dtype}, got {list(x.shape)} of "
                           f"{x.dtype}")


def glr_forward(gates, c0=None, lengths=None, *, training=False, out=None):
    """``(h, cT, marks)`` without autograd. ``marks`` is what
    ``glr_backward`` needs of the forward pass, None unless ``training``.
    ``out``: a contiguous [T, B, H] to write ``h`` into."""
    if not _eager(gates):
        return _C.ext().glr_forward(gates, c0, lengths, training, out)
    _check_eager("glr_forward", gates, 3, c0=c0)
    _check_lengths("glr_forward", gates, lengths)
    _check_like_h("glr_forward", "out", out, gates, gates.size(2) // 4)
    with torch.no_grad():
        h, cT = F_ref.glr_layer(gates, c0, lengths)
    if out is not None:
        h = out.copy_(h)
    return h, cT, None


def glr_backward(dh, dcT, gates, c0, marks, lengths=None, *, out=None):
    """``(dgates, dc0)`` from the gradients of ``h`` and ``cT`` (either may
    be None), the forward pass's inputs and its ``marks``. ``out``: a
    contiguous tensor like ``gates`` to write ``dgates`` into."""
    if not _eager(gates):
        if marks is None:
            raise RuntimeError("glr_backward: marks must be what "
                               "glr_forward(training=True) returned for "
                               "these gates")
        return _C.ext().glr_backward(dh, dcT, gates, c0, marks, lengths, out)
    _check_eager("glr_backward", gates, 3, c0=c0, dcT=dcT)
    _check_lengths("glr_backward", gates, lengths)
    _check_like_h("glr_backward", "dh", dh, gates, gates.size(2) // 4)
    _check_like_h("glr_backward", "out", out, gates, gates.size(2))
    with torch.enable_grad():
        g = gates.detach().requires_grad_()
        c = (torch.zeros(gates.size(1), gates.size(2) // 4,
                         device=gates.device) if c0 is None
             else c0.detach().clone()).requires_grad_()
        h, cT = F_ref.glr_layer(g, c, lengths)
        dh = torch.zeros_like(h) if dh is None else dh
        dcT = torch.zeros_like(cT) if dcT is None else dcT
        ends = ((h, dh), (cT, dcT))[gates.size(0) == 0:]  # no steps, no h
        dg, dc0 = torch.autograd.grad([x for x, _ in ends], (g, c),
                                      [d for _, d in ends],
                                      allow_unused=True)
    dg = torch.zeros_like(g) if dg is None else dg
    return (dg if out is None else out.copy_(dg)), dc0


def glr_step(gates, c):
    """One token: ``h`` [B, H] from ``gates`` [B, 4H]; the state ``c``
    (float32 [B, H], rows may be apart) is advanced in place. Has no
    backward pass: call it under ``torch.no_grad()``."""
    if not _eager(gates):
        return _C.ext().glr_step(gates, c)
    if torch.is_grad_enabled() and (gates.requires_grad or c.requires_grad):
        raise RuntimeError("glr_step: has no backward pass; call it under "
                           "torch.no_grad(), or use glr()")
    _check_eager("glr_step", gates, 2, c=c)
    h, new = F_ref.glr_step(gates, c)
    c.copy_(new)
    return h


class GlrFn(torch.autograd.Function):
    """The kernels under autograd; no second derivative."""

    @staticmethod
    def forward(ctx, gates, c0, lengths):
        ctx.set_materialize_grads(False)
        h, cT, marks = _C.ext().glr_forward(gates, c0, lengths, True, None)
        ctx.save_for_backward(gates, c0, lengths, marks)
        return h, cT

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dcT):
        gates, c0, lengths, marks = ctx.saved_tensors
        if dh is None and dcT is None:
            return None, None, None
        dgates, dc0 = _C.ext().glr_backward(dh, dcT, gates, c0, marks,
                                            lengths, None)
        return dgates, (dc0 if ctx.needs_input_grad[1] else None), None


def glr(gates, c0=None, lengths=None):
    """``(h, cT)``, differentiable in ``gates`` and ``c0``: once, and on the
    GPU in reverse mode only (a tensor with a tangent is refused)."""
    if not _eager(gates):
        if torch.is_grad_enabled() and (
                gates.requires_grad or (c0 is not None and c0.requires_grad)):
            return GlrFn.apply(gates, c0, lengths)
        return _C.ext().glr_forward(gates, c0, lengths, False, None)[:2]
    _check_eager("glr", gates, 3, c0=c0)
    _check_lengths("glr", gates, lengths)
    return F_ref.glr_layer(gates, c0, lengths)
