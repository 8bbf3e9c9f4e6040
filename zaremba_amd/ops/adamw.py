"""AdamW over many tensors at once, with the global gradient norm clipped.

    g = grad * grad_scale * min(1, max_norm / (|grad| * grad_scale + 1e-6))
    m = b1 m + (1 - b1) g        v = b2 v + (1 - b2) g^2
    p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v / (1 - b2^t)) + eps)

The clip is the one of the SGD step (reference main.py:115); the decay is
decoupled and applies to every tensor of the call.

States in 32 bits are ``m`` and ``v``. States in 8 bits are blocks of 256
e4m3 codes with one float32 scale each: of ``m``, and of ``r = sqrt(v)``. A
value is its code times its scale. The codes of ``m`` are the nearest ones;
those of ``r`` are drawn from the two neighbours so that ``v`` is right in
the mean (an average over 1 / (1 - b2) steps moves by far less than half a
code a step, and would stand still), with a hash of the step and the place in
the tensor: the same inputs give the same states. A block whose largest
magnitude is under 2^-100 is stored as zeros. A gradient that is not finite
makes the norm, and with it the update, not finite, as it does in SGD.

On the GPU this is two launches for each 48 tensors, on the current stream
of the parameters' device; the step count lives on the device, so that a
captured step may be replayed. On the CPU (or with ZAREMBA_AMD_FORCE_EAGER=1)
the eager math of ops/functional.py runs.
"""

from __future__ import annotations

import torch

from .. import _C
from . import functional as F_ref

E4M3 = torch.float8_e4m3fn
BLOCK = 256
LEAST_EPS = torch.finfo(torch.float32).tiny


def _check(lr, betas, eps, weight_decay, max_norm, grad_scale=1.0):
    if not lr >= 0:
        raise ValueError(f"adamw_step_: lr must not be negative, got {lr}")
    if not (0 <= betas[0] < 1 and 0 <= betas[1] < 1):
        raise ValueError(f"adamw_step_: betas must be in [0, 1), got {betas}")
    if not eps >= LEAST_EPS:
        # a smaller one is 0 in float32, or 1 / eps is not finite there: a
        # value that has seen no gradient would become 0 * inf
        raise ValueError("adamw_step_: eps must be positive, and at least "
                         f"{LEAST_EPS:.3g}, got {eps}")
    if not weight_decay >= 0:
        raise ValueError("adamw_step_: weight_decay must not be negative, "
                         f"got {weight_decay}")
    if max_norm is not None and not max_norm > 0:
        raise ValueError("adamw_step_: max_norm must be positive or None, "
                         f"got {max_norm}")
    if not grad_scale > 0:
        raise ValueError("adamw_step_: grad_scale must be positive, got "
                         f"{grad_scale}")


def _check_lists(params, grads, exp_avgs, exp_avg_sqs, step, m_scales,
                 v_scales, shadows):
    """What the eager math cannot do, before anything is written; the
    kernels' host side has checks of its own."""
    def check(ok, what):
        if not ok:
            raise RuntimeError(f"adamw_step_: {what}")

    bits8 = len(exp_avgs) > 0 and exp_avgs[0].dtype == E4M3
    check(bits8 == (m_scales is not None) == (v_scales is not None),
          "states in 8 bits need exp_avg_scales and exp_avg_sq_scales, "
          "states in 32 bits have none")
    lists = {"grads": grads, "exp_avgs": exp_avgs, "exp_avg_sqs": exp_avg_sqs,
             "exp_avg_scales": m_scales, "exp_avg_sq_scales": v_scales,
             "shadows": shadows, "params": params}
    lists = {name: x for name, x in lists.items() if x is not None}
    check(all(len(x) == len(params) for x in lists.values()),
          "the lists differ in length")
    check(step.dtype == torch.int64 and step.numel() == 1,
          "step must be one int64")
    written = [step]
    for name, tensors in lists.items():
        for k, x in enumerate(tensors):
            if x is None and name == "shadows":
                continue
            n = params[k].numel()
            n = -(-n // BLOCK) if name.endswith("scales") else n
            check(x.numel() == n, f"{name}[{k}] has {x.numel()} values, "
                  f"expected {n}")
            # the eager math reads gradients, and writes copies, of any order
            check(name in ("grads", "shadows") or x.is_contiguous(),
                  f"{name}[{k}] must be contiguous")
            if n and name != "grads":
                written.append(x)
    check(len({x.data_ptr() for x in written}) == len(written),
          "parameters, states or shadows share memory")


@torch.no_grad()
def adamw_step_(params, grads, exp_avgs, exp_avg_sqs, step, *, lr,
                betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01,
                max_norm=None, grad_scale=1.0, exp_avg_scales=None,
                exp_avg_sq_scales=None, shadows=None):
    """One step, in place. Lists of contiguous tensors on one device:

    ``params``: float32 masters. ``grads``: float32 or bfloat16.
    ``exp_avgs``, ``exp_avg_sqs``: float32, or float8_e4m3fn with the lists
    of scales (float32, ceil(n / 256) each). ``shadows``: bfloat16 copies of
    the parameters to rewrite in the same pass, None where there is none.
    ``step``: one int64 on the device, the steps done before; advanced.

    Returns the gradient norm before the clip (0-d float32), None where
    ``max_norm`` is None: nothing is clipped then, and no norm computed.
    """
    _check(lr, betas, eps, weight_decay, max_norm, grad_scale)
    if len(params) == 0:
        raise RuntimeError("adamw_step_: no parameters")
    if params[0].is_cuda and not _C.force_eager_env():
        return _C.ext().adamw_step_(
            params, grads, exp_avgs, exp_avg_sqs, step, lr, betas[0],
            betas[1], eps, weight_decay, max_norm, grad_scale,
            exp_avg_scales, exp_avg_sq_scales, shadows)
    _check_lists(params, grads, exp_avgs, exp_avg_sqs, step, exp_avg_scales,
                 exp_avg_sq_scales, shadows)
    return F_ref.adamw_step_(
        params, grads, exp_avgs, exp_avg_sqs, step, lr, betas, eps,
        weight_decay, max_norm, grad_scale, exp_avg_scales,
        exp_avg_sq_scales, shadows)


class AdamW:
    """The states of a model's parameters, in the order of
    ``model.parameters()``. ``trainer.adamw_step`` makes the step; on the HIP
    engine it is what rewrites the bf16 shadows, too, that the next forward
    reads, so ``step`` alone is for parameters without shadows."""

    def __init__(self, params, betas=(0.9, 0.999), eps=1e-8,
                 weight_decay=0.01, bits=32):
        if bits not in (8, 32):
            raise ValueError(f"AdamW: states have 8 or 32 bits, got {bits}")
        _check(0.0, betas, eps, weight_decay, None)
        self.params = list(params)
        if not self.params:
            raise ValueError("AdamW: no parameters")
        self.betas, self.eps = tuple(betas), eps
        self.weight_decay, self.bits = weight_decay, bits
        dev = self.params[0].device
        kind = E4M3 if bits == 8 else torch.float32
        zeros = lambda: [  # noqa: E731
            torch.zeros(p.shape, dtype=torch.uint8 if bits == 8 else kind,
                        device=dev).view(kind) for p in self.params]
        scales = lambda: [  # noqa: E731
            torch.zeros(-(-p.numel() // BLOCK), device=dev)
            for p in self.params] if bits == 8 else None
        self.exp_avgs, self.exp_avg_sqs = zeros(), zeros()
        self.exp_avg_scales, self.exp_avg_sq_scales = scales(), scales()
        self.step_count = torch.zeros(1, dtype=torch.int64, device=dev)

    def step(self, lr, max_norm=None, grad_scale=1.0, shadow_of=None):
        """Updates the parameters that have a gradient. ``shadow_of``: bf16
        copies by ``id(parameter)``."""
        at = [k for k, p in enumerate(self.params) if p.grad is not None]
        if not at:
            raise RuntimeError("AdamW: no parameter has a gradient")
        pick = lambda x: None if x is None else [x[k] for k in at]  # noqa
        params = [self.params[k].detach() for k in at]
        return adamw_step_(
            params, [self.params[k].grad for k in at], pick(self.exp_avgs),
            pick(self.exp_avg_sqs), self.step_count, lr=lr, betas=self.betas,
            eps=self.eps, weight_decay=self.weight_decay, max_norm=max_norm,
            grad_scale=grad_scale, exp_avg_scales=pick(self.exp_avg_scales),
            exp_avg_sq_scales=pick(self.exp_avg_sq_scales),
            shadows=None if shadow_of is None else
            [shadow_of.get(id(self.params[k])) for k in at])

    _LISTS = ("exp_avgs", "exp_avg_sqs", "exp_avg_scales",
              "exp_avg_sq_scales")

    def state_dict(self):
        """A copy on the CPU, which later steps leave as it is."""
        copy = lambda t: t.to("cpu", copy=True)  # noqa: E731
        out = {"bits": self.bits, "step_count": copy(self.step_count)}
        for name in self._LISTS:
            x = getattr(self, name)
            out[name] = None if x is None else [copy(t) for t in x]
        return out

    def load_state_dict(self, state):
        if state["bits"] != self.bits:
            raise ValueError(f"AdamW: the saved states have {state['bits']} "
                             f"bits, these {self.bits}")
        names = [name for name in self._LISTS
                 if getattr(self, name) is not None]
        for name in names:  # all of them, before one is written
            if ([t.shape for t in getattr(self, name)]
                    != [t.shape for t in state[name]]):
                raise ValueError(f"AdamW: the saved {name} are of another "
                                 "model")
        for name in names:
            for a, b in zip(getattr(self, name), state[name]):
                a.copy_(b)
        self.step_count.copy_(state["step_count"])
