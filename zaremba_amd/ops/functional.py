"""Eager (pure-PyTorch) implementations of every op in the framework.

These are the semantic ground truth: the math transcribes the reference
implementation exactly (citations per function), in a numerically stable
form where the reference is naive. They serve three roles:

  1. the CPU execution path (config 1: plumbing, no GPU),
  2. the fp32 oracle that every HIP kernel is unit-tested against,
  3. the fallback when running on non-gfx950 devices for debugging.

The HIP kernel path lives in zaremba_amd/ops/hip_ops.py + csrc/.
"""

from __future__ import annotations

from typing import List, Optional, Tuple

import torch


# ---------------------------------------------------------------------------
# LSTM cell (reference model.py:34-45; gate order i, f, o, n)
# ---------------------------------------------------------------------------

def lstm_step(
    x: torch.Tensor,
    h: torch.Tensor,
    c: torch.Tensor,
    W_x: torch.Tensor,
    W_h: torch.Tensor,
    b_x: torch.Tensor,
    b_h: torch.Tensor,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """One LSTM timestep, gate order (input, forget, output, new).

    Note this differs from nn.LSTM's (i, f, g, o) order — state_dicts are
    not interchangeable between implementations (reference model.py:37-41).
    """
    gx = torch.addmm(b_x, x, W_x.t())
    gh = torch.addmm(b_h, h, W_h.t())
    xi, xf, xo, xn = gx.chunk(4, 1)
    hi, hf, ho, hn = gh.chunk(4, 1)
    i = torch.sigmoid(xi + hi)
    f = torch.sigmoid(xf + hf)
    o = torch.sigmoid(xo + ho)
    n = torch.tanh(xn + hn)
    c = f * c + i * n
    h = o * torch.tanh(c)
    return h, c


def lstm_layer(
    x: torch.Tensor,
    h0: torch.Tensor,
    c0: torch.Tensor,
    W_x: torch.Tensor,
    W_h: torch.Tensor,
    b_x: torch.Tensor,
    b_h: torch.Tensor,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Unrolled LSTM layer over a [T, B, X] input (reference model.py:48-55)."""
    h, c = h0, c0
    outputs = []
    for x_t in x.unbind(0):
        h, c = lstm_step(x_t, h, c, W_x, W_h, b_x, b_h)
        outputs.append(h)
    return torch.stack(outputs), h, c


# ---------------------------------------------------------------------------
# Gated linear recurrence: the same cell without its recurrent product
# ---------------------------------------------------------------------------

def glr_step(gates: torch.Tensor, c: torch.Tensor
             ) -> Tuple[torch.Tensor, torch.Tensor]:
    """One step from [B, 4H] pre-activations, gate order (i, f, o, n), in
    the state's type (float32 or wider); h in the gates' type."""
    i, f, o, n = gates.to(c.dtype).chunk(4, 1)
    c = torch.sigmoid(f) * c + torch.sigmoid(i) * torch.tanh(n)
    return (torch.sigmoid(o) * torch.tanh(c)).to(gates.dtype), c


def glr_layer(gates: torch.Tensor, c0: Optional[torch.Tensor] = None,
              lengths: Optional[torch.Tensor] = None
              ) -> Tuple[torch.Tensor, torch.Tensor]:
    """The recurrence over [T, B, 4H]; row b ends after lengths[b] steps."""
    T, B, H = gates.size(0), gates.size(1), gates.size(2) // 4
    c = c0
    if c is None:
        wide = gates.dtype if gates.dtype == torch.float64 else torch.float32
        c = torch.zeros(B, H, dtype=wide, device=gates.device)
    if T == 0:
        return gates.new_empty(0, B, H), c.clone()
    outputs = []
    for t, g in enumerate(gates.unbind(0)):
        if lengths is not None:
            live = (t < lengths)[:, None]
            # what stands in a finished row must not reach a gradient
            g = torch.where(live, g, torch.zeros_like(g))
            h, new = glr_step(g, c)
            h = torch.where(live, h, torch.zeros_like(h))
            c = torch.where(live, new, c)
        else:
            h, c = glr_step(g, c)
        outputs.append(h)
    return torch.stack(outputs), c


# ---------------------------------------------------------------------------
# Embedding (reference model.py:6-17)
# ---------------------------------------------------------------------------

def embedding(W: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
    """[T,B] int64 -> [T,B,H] gather from the [V,H] table."""
    return W[x]


# ---------------------------------------------------------------------------
# Output projection (reference model.py:57-71)
# ---------------------------------------------------------------------------

def linear(x: torch.Tensor, W: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """Flattens [T,B,H] -> [T*B,H]; returns 2-D [T*B, V] scores."""
    return torch.addmm(b, x.view(-1, x.size(-1)), W.t())


# ---------------------------------------------------------------------------
# Loss (reference main.py:77-84)
# ---------------------------------------------------------------------------

def nll_loss(scores: torch.Tensor, y: torch.Tensor) -> torch.Tensor:
    """batch_size x cross-entropy: sums over batch, averages over time.

    The reference computes a numerically naive softmax (exp then
    normalize, main.py:79-80) which overflows outside fp32; this is the
    same math through a max-subtracted log-softmax. Scale convention:
    mean over the T*B tokens of (-log p) times B, i.e. the per-timestep
    loss is summed over the batch and averaged over time (main.py:82-84).
    """
    batch_size = y.size(1)
    logp = torch.log_softmax(scores.float(), dim=1)
    answer_logp = logp[torch.arange(y.numel(), device=y.device), y.reshape(-1)]
    return torch.mean(-answer_logp * batch_size)


def ensemble_nll_loss(scores_list: List[torch.Tensor], y: torch.Tensor) -> torch.Tensor:
    """NLL of the arithmetic mean of per-model probabilities
    (reference ensemble.py:97-109), via stable softmax."""
    batch_size = y.size(1)
    probs = torch.stack([torch.softmax(s.float(), dim=1) for s in scores_list])
    mean_probs = probs.mean(dim=0)
    answer = mean_probs[torch.arange(y.numel(), device=y.device), y.reshape(-1)]
    return torch.mean(-torch.log(answer) * batch_size)


# ---------------------------------------------------------------------------
# Optimizer step (reference main.py:115-117)
# ---------------------------------------------------------------------------

def clip_grad_and_sgd_(
    params: List[torch.Tensor], max_norm: float, lr: float
) -> torch.Tensor:
    """Global L2 grad-norm clip followed by vanilla SGD, in place.

    Matches torch.nn.utils.clip_grad_norm_ + the reference's manual
    ``param -= lr * param.grad`` (main.py:115-117). Returns the
    pre-clip total norm (the value the reference logs as dw.norm()).
    """
    grads = [p.grad for p in params if p.grad is not None]
    total_norm = torch.norm(torch.stack([torch.norm(g.detach(), 2.0) for g in grads]), 2.0)
    clip_coef = max_norm / (total_norm + 1e-6)
    coef = torch.clamp(clip_coef, max=1.0)
    with torch.no_grad():
        for p in params:
            if p.grad is not None:
                p.add_(p.grad, alpha=-lr * float(coef))
    return total_norm


# ---------------------------------------------------------------------------
# AdamW, states in 32 or in 8 bits (ops/adamw.py says what they are)
# ---------------------------------------------------------------------------

_E4M3_MAX, _TINY = 448.0, 2.0 ** -100


def _blocks(x: torch.Tensor) -> torch.Tensor:
    """[ceil(n / 256), 256] of the values, zeros behind the last."""
    x = x.reshape(-1)
    return torch.nn.functional.pad(x, (0, -x.numel() % 256)).view(-1, 256)


def _e4m3_scales(x: torch.Tensor):
    amax = x.abs().amax(1)
    empty = amax < _TINY
    zero = torch.zeros_like(amax)
    return (torch.where(empty, zero, amax * (1 / _E4M3_MAX)),
            torch.where(empty, zero, amax.reciprocal() * _E4M3_MAX)[:, None])


def hash_uniform(index: torch.Tensor, step) -> torch.Tensor:
    """Numbers in [0, 1) with 24 bits, from a 32-bit mixing hash
    (csrc/adamw.hip names it)."""
    low = 0xFFFFFFFF
    x = (index.long() * 0x9E3779B1 + step * 0x85EBCA77) & low
    x = ((x ^ (x >> 16)) * 0x7FEB352D) & low
    x = ((x ^ (x >> 15)) * 0x846CA68B) & low
    return ((x ^ (x >> 16)) >> 8).float() * 2.0 ** -24


def draw_e4m3(x: torch.Tensor, u: torch.Tensor) -> torch.Tensor:
    """Codes (uint8) of one of the two e4m3 values beside x >= 0, the upper
    one where u < (x^2 - a^2) / (b^2 - a^2); 0 only for 0."""
    x = x.clamp(max=_E4M3_MAX)
    low = torch.where(x < 2.0 ** -6, (x * 512).int(),
                      (x.view(torch.int32) >> 20) - 960).clamp(0, 126)
    value = lambda c: c.to(torch.uint8).view(  # noqa: E731
        torch.float8_e4m3fn).float()
    a, b = value(low), value((low + 1).clamp(max=126))
    up = u * (b * b - a * a) < x * x - a * a
    return (low + torch.where(low == 0, x > 0, up)).clamp(
        max=126).to(torch.uint8)


def adamw_step_(params, grads, exp_avgs, exp_avg_sqs, step, lr, betas, eps,
                weight_decay, max_norm, grad_scale, exp_avg_scales,
                exp_avg_sq_scales, shadows):
    step += 1
    t = int(step)
    b1, b2 = betas
    norm, scale = None, grad_scale
    if max_norm is not None:
        norm = torch.stack([g.double().square().sum() for g in grads]
                           ).sum().sqrt() * grad_scale
        scale = grad_scale * float(torch.clamp(max_norm / (norm + 1e-6),
                                               max=1.0))
        norm = norm.float()
    rate, root = lr / (1 - b1 ** t), (1 - b2 ** t) ** -0.5
    for k, p in enumerate(params):
        n = p.numel()
        g = grads[k].reshape(-1).float() * scale
        if exp_avg_scales is None:
            m, v = exp_avgs[k].view(-1), exp_avg_sqs[k].view(-1)
        else:
            m = (_blocks(exp_avgs[k].float())
                 * exp_avg_scales[k][:, None]).view(-1)[:n]
            v = (_blocks(exp_avg_sqs[k].float())
                 * exp_avg_sq_scales[k][:, None]).view(-1)[:n].square()
        m = m * b1 + g * (1 - b1)
        v = v * b2 + g * g * (1 - b2)
        r = v.sqrt()
        flat = p.view(-1)
        flat.copy_(flat * (1 - lr * weight_decay)
                   - rate * (m / (r * root + eps)))
        if shadows is not None and shadows[k] is not None:
            shadows[k].copy_(p)
        if exp_avg_scales is None:
            exp_avgs[k].view(-1).copy_(m)
            exp_avg_sqs[k].view(-1).copy_(v)
            continue
        mb, rb = _blocks(m), _blocks(r)
        scales, inv = _e4m3_scales(mb)
        exp_avg_scales[k].copy_(scales)
        exp_avgs[k].copy_((mb * inv).view(-1)[:n].to(torch.float8_e4m3fn)
                          .view(p.shape))
        scales, inv = _e4m3_scales(rb)
        exp_avg_sq_scales[k].copy_(scales)
        u = hash_uniform(torch.arange(n, device=p.device), t)
        codes = draw_e4m3((rb * inv).view(-1)[:n], u)
        exp_avg_sqs[k].copy_(codes.view(torch.float8_e4m3fn).view(p.shape))
    return norm
