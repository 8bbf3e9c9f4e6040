"""What the gated linear recurrence and the AdamW step are measured on.

Each case is one call, or one pair of calls, that a training or evaluation
program makes. ``run`` computes a case in its plain form (elementary torch
operations in 32 bits) where ``own`` is false, and through
``zaremba_amd.ops`` where it is true.

Gated linear recurrence, for pre-activations ``(i, f, o, n)`` of a time step:

    c_t = sigmoid(f_t) c_{t-1} + sigmoid(i_t) tanh(n_t)
    h_t = sigmoid(o_t) tanh(c_t)

A row of the batch whose length is over keeps its state, and its ``h`` is zero.

AdamW over many tensors, with the global gradient norm clipped:

    g = grad * min(1, max_norm / (|grad| + 1e-6))
    m = b1 m + (1 - b1) g          v = b2 v + (1 - b2) g^2
    p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v / (1 - b2^t)) + eps)

States in 8 bits are blocks of 256 values: e4m3 codes and one 32-bit scale a
block, of m and of r = sqrt(v). The codes of m are the nearest. Those of r are
drawn from its two neighbours, so that v is right in the mean: an average over
1000 steps moves by less than half a code a step, and would stand still. What
is drawn with is a hash of the step and the place in the tensor. A root that is
not zero is never rounded to zero.
"""

import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BETAS, EPS, DECAY = (0.9, 0.999), 1e-8, 0.01
BLOCK = 256
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
TINY = 2.0 ** -100  # a block that is smaller throughout is stored as zeros

MOST_STEPS = 65536 * 1500       # channel steps of the largest recurrence
MOST_PARAMS = 66_022_000        # parameters of the largest update


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # one token for each of 20 streams of the small model (hidden 200)
        dict(name="step small", op="step", T=1, B=20, H=200, type="bf16",
             ragged=False, batch_first=False),
        # one token for each of 512 streams of the large model (hidden 1500)
        dict(name="step many", op="step", T=1, B=512, H=1500, type="bf16",
             ragged=False, batch_first=False),
        # one evaluation window of the large model
        dict(name="forward window", op="forward", T=35, B=20, H=1500,
             type="bf16", ragged=False, batch_first=False),
        # one training window of a layer of the large model
        dict(name="train window", op="train", T=35, B=20, H=1500,
             type="bf16", ragged=False, batch_first=False),
        # one training window of the medium model in full precision
        dict(name="train window fp32", op="train", T=35, B=20, H=650,
             type="fp32", ragged=False, batch_first=False),
        # padded sentences, batch first, odd sizes
        dict(name="train ragged", op="train", T=1001, B=17, H=651,
             type="fp16", ragged=True, batch_first=True),
        # a validation text scored as one stream
        dict(name="forward long", op="forward", T=65536, B=1, H=1500,
             type="bf16", ragged=False, batch_first=False),
        # training on one unbroken text
        dict(name="train long", op="train", T=65536, B=1, H=1500,
             type="bf16", ragged=False, batch_first=False),
        # the small model's update
        dict(name="adamw small", op="adamw", shapes="model", hidden=200,
             vocab=10000, layers=2, bits=32, grad="fp32", shadow=True),
        # the large model's update
        dict(name="adamw large", op="adamw", shapes="model", hidden=1500,
             vocab=10000, layers=2, bits=32, grad="fp32", shadow=True),
        # the same with states in 8 bits
        dict(name="adamw large 8 bit", op="adamw", shapes="model",
             hidden=1500, vocab=10000, layers=2, bits=8, grad="fp32",
             shadow=True),
        # many tensors of odd sizes, gradients in bf16, states in 8 bits
        dict(name="adamw odd 8 bit", op="adamw", shapes="odd", tensors=48,
             params=9_000_001, bits=8, grad="bf16", shadow=False),
    ]


def _spread(rng, low, high):
    """A whole number, even over its logarithm."""
    return min(high, max(low, int(round(math.exp(
        rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["step", "forward", "train", "train", "adamw", "adamw"])
    if op == "adamw":
        bits, grad = rng.choice([8, 32]), rng.choice(["fp32", "bf16"])
        shadow = rng.random() < 0.5
        if rng.random() < 0.5:
            return dict(op=op, shapes="model", hidden=_spread(rng, 200, 1500),
                        vocab=_spread(rng, 1000, 10000),
                        layers=rng.randint(1, 2), bits=bits, grad=grad,
                        shadow=shadow)
        tensors = _spread(rng, 1, 200)
        return dict(op=op, shapes="odd", tensors=tensors,
                    params=_spread(rng, 1000 * tensors, MOST_PARAMS),
                    bits=bits, grad=grad, shadow=shadow)
    T = 1 if op == "step" else _spread(rng, 2, 65536)
    H = _spread(rng, 100, 2048)
    B = _spread(rng, 1, max(1, min(512, MOST_STEPS // (T * H))))
    T = min(T, MOST_STEPS // (B * H))
    return dict(op=op, T=T, B=B, H=H, type=rng.choice(sorted(TYPES)),
                ragged=op != "step" and rng.random() < 0.4,
                batch_first=op != "step" and rng.random() < 0.4)


def _sizes(case):
    if case["shapes"] == "model":
        h, v = case["hidden"], case["vocab"]
        layer = [4 * h * h, 4 * h * h, 4 * h, 4 * h]
        return [v * h] + layer * case["layers"] + [v * h, v]
    # sizes of a broken stick, whose pieces differ by orders of magnitude
    n, total = case["tensors"], case["params"]
    parts = np.random.RandomState(n).lognormal(0.0, 2.0, n)
    sizes = [max(1, int(total * p / parts.sum())) for p in parts]
    sizes[int(np.argmax(parts))] += max(0, total - sum(sizes))
    return sizes


def work(case):
    if case["op"] == "adamw":
        n = sum(_sizes(case))
        # read p, g, m, v; write p, m, v and the shadow
        state = 16 if case["bits"] == 32 else 4 + 4 * 4 / BLOCK
        each = (8 + (4 if case["grad"] == "fp32" else 2) + state
                + (2 if case["shadow"] else 0))
        return {"bytes": n * each, "flops": n * 18}
    T, B, H = case["T"], case["B"], case["H"]
    e = TYPES[case["type"]].itemsize
    n = T * B * H
    if case["op"] == "train":
        # forward: gates in, h out; backward: gates and dh in, dgates out
        return {"bytes": n * e * 14 + B * H * 20, "flops": n * 75}
    return {"bytes": n * e * 5 + B * H * 8, "flops": n * 25}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _time_major(case, gen, width, scale, type_):
    """[T, B, width], stored batch first where the case says so."""
    T, B = case["T"], case["B"]
    shape = (B, T, width) if case["batch_first"] else (T, B, width)
    x = torch.randn(shape, generator=gen, device=DEVICE).mul_(scale).to(type_)
    return x.transpose(0, 1) if case["batch_first"] else x


def _prepare_recurrence(case, gen):
    T, B, H = case["T"], case["B"], case["H"]
    type_ = TYPES[case["type"]]
    s = {"gates": _time_major(case, gen, 4 * H, 1.5, type_),
         "c0": torch.randn(B, H, generator=gen, device=DEVICE),
         "lengths": None}
    if case["ragged"]:
        lengths = torch.randint(1, T + 1, (B,), generator=gen, device=DEVICE)
        lengths[-1] = T
        if B > 2:
            lengths[0] = 0  # a row of padding only
        s["lengths"] = lengths.to(torch.int32)
    if case["op"] == "train":
        s["dh"] = _time_major(case, gen, H, 1.0, type_)
        s["dcT"] = torch.randn(B, H, generator=gen, device=DEVICE)
    return s


def _quantise(x, amax):
    """Codes and scales of [blocks, BLOCK] values whose magnitudes end at amax."""
    empty = amax < TINY
    scale = torch.where(empty, torch.zeros_like(amax), amax / E4M3_MAX)
    inv = torch.where(empty, torch.zeros_like(amax), E4M3_MAX / amax)
    return (x * inv[:, None]).to(E4M3), scale


def _uniform(index, step):
    """Numbers in [0, 1) for places of a tensor: a 32-bit mixing hash."""
    x = (index.long() * 0x9E3779B1 + step * 0x85EBCA77) & 0xFFFFFFFF
    x = ((x ^ (x >> 16)) * 0x7FEB352D) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x846CA68B) & 0xFFFFFFFF
    return ((x ^ (x >> 16)) >> 8).float() * 2.0 ** -24


def _quantise_root(r, index, step):
    amax = r.amax(1)
    empty = amax < TINY
    scale = torch.where(empty, torch.zeros_like(amax), amax / E4M3_MAX)
    inv = torch.where(empty, torch.zeros_like(amax), E4M3_MAX / amax)
    x = (r * inv[:, None]).clamp(max=E4M3_MAX)
    # the code below: 3 bits of the mantissa, or 512ths under 2^-6
    low = torch.where(x < 2.0 ** -6, (x * 512).int(),
                      (x.view(torch.int32) >> 20) - 960)
    value = low.to(torch.uint8).view(E4M3).float()
    above = (low + 1).clamp(max=126).to(torch.uint8).view(E4M3).float()
    up = _uniform(index, step).view(x.shape) * (
        above * above - value * value) < x * x - value * value
    up = torch.where(low == 0, x > 0, up)
    codes = (low + up).clamp(max=126).to(torch.uint8)
    return codes.view(E4M3), scale


def _prepare_adamw(case, gen):
    sizes = _sizes(case)
    starts, at = [], 0
    for n in sizes:  # each tensor begins on a block of its own
        starts.append(at)
        at += -(-n // BLOCK) * BLOCK
    place = torch.full((at,), -1, dtype=torch.int32, device=DEVICE)
    for a, n in zip(starts, sizes):
        place[a:a + n] = torch.arange(n, device=DEVICE)
    live = place >= 0

    def flat(scale):
        return torch.randn(at, generator=gen, device=DEVICE).mul_(
            scale).mul_(live)

    # gradients and their averages span orders of magnitude between blocks;
    # the gradient's norm is twice what it is clipped to
    spread = torch.exp2(torch.randn(at // BLOCK, 1, generator=gen,
                                    device=DEVICE) * 2)
    max_norm = 5.0
    g = (flat(1.0).view(-1, BLOCK) * spread).view(-1)
    unit = max_norm / g.norm()
    s = {"p": flat(0.04), "g": (g * (2 * unit)).to(TYPES[case["grad"]]),
         "place": place}
    m = flat(0.3).view(-1, BLOCK) * spread * unit
    v = (flat(1.0).view(-1, BLOCK) * spread * unit).square()
    if case["bits"] == 32:
        s["m"], s["v"] = m.view(-1), v.view(-1)
        s["ms"] = s["vs"] = None
    else:
        codes, s["ms"] = _quantise(m, m.abs().amax(1))
        s["m"] = codes.view(-1)
        codes, s["vs"] = _quantise_root(v.sqrt(), place, 1000)
        s["v"] = codes.view(-1)
    s["shadow"] = s["p"].to(torch.bfloat16) if case["shadow"] else None
    s["step"] = torch.full((1,), 1000, dtype=torch.int64, device=DEVICE)
    s["lr"], s["max_norm"] = 1e-3, max_norm

    def views(x):
        return [x[a:a + n] for a, n in zip(starts, sizes)]

    def block_views(x):
        return [x[a // BLOCK:a // BLOCK + -(-n // BLOCK)]
                for a, n in zip(starts, sizes)]

    s["lists"] = {k: views(s[k]) for k in ("p", "g", "m", "v")}
    s["lists"]["shadow"] = views(s["shadow"]) if case["shadow"] else None
    for k in ("ms", "vs"):
        s["lists"][k] = block_views(s[k]) if case["bits"] == 8 else None
    return s


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    if case["op"] == "adamw":
        s = _prepare_adamw(case, gen)
    else:
        s = _prepare_recurrence(case, gen)
        if case["op"] == "step":
            s["gates"] = s["gates"][0]
    s["op"], s["bits"] = case["op"], case.get("bits")
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------

def _scan(a, b):
    """x_t = a_t x_{t-1} + b_t over the first axis, by doubling."""
    d = 1
    while d < a.size(0):
        b = torch.cat([b[:d], b[d:] + a[d:] * b[:-d]])
        a = torch.cat([a[:d], a[d:] * a[:-d]])
        d *= 2
    return b


def _live(s, T):
    t = torch.arange(T, device=s["gates"].device)
    return (t[:, None] < s["lengths"][None, :])[..., None]


def _plain_recurrence(s, backward):
    gates, c0 = s["gates"], s["c0"]
    i, f, o, n = gates.float().chunk(4, -1)
    i, f, o, n = torch.sigmoid(i), torch.sigmoid(f), torch.sigmoid(o), \
        torch.tanh(n)
    a, b = f, i * n
    if s["lengths"] is not None:
        live = _live(s, gates.size(0))
        a = torch.where(live, a, torch.ones_like(a))
        b = torch.where(live, b, torch.zeros_like(b))
    first = torch.cat([(a[:1] * c0 + b[:1]), b[1:]])
    c = _scan(a, first)
    tc = torch.tanh(c)
    h = o * tc
    if s["lengths"] is not None:
        h = torch.where(live, h, torch.zeros_like(h))
    out = {"h": h.to(gates.dtype), "cT": c[-1]}
    if not backward:
        return out
    dh = s["dh"].float()
    u = dh * o * (1 - tc * tc)
    if s["lengths"] is not None:
        u = torch.where(live, u, torch.zeros_like(u))
    u = torch.cat([u[:-1], u[-1:] + s["dcT"]])
    later = torch.cat([a[1:], torch.ones_like(a[:1])])
    g = _scan(later.flip(0), u.flip(0)).flip(0)
    before = torch.cat([c0[None], c[:-1]])
    d = torch.cat([g * n * i * (1 - i), g * before * f * (1 - f),
                   dh * tc * o * (1 - o), g * i * (1 - n * n)], -1)
    if s["lengths"] is not None:
        d = torch.where(live, d, torch.zeros_like(d))
    out["dgates"] = d.to(gates.dtype)
    out["dc0"] = a[0] * g[0]
    return out


def _plain_step(s):
    i, f, o, n = s["gates"].float().chunk(4, -1)
    c = torch.sigmoid(f) * s["c0"] + torch.sigmoid(i) * torch.tanh(n)
    s["c0"].copy_(c)
    return {"h": (torch.sigmoid(o) * torch.tanh(c)).to(s["gates"].dtype),
            "c": s["c0"]}


def _plain_adamw(s):
    b1, b2 = BETAS
    s["step"] += 1
    t = s["step"].double()
    norm = s["g"].double().square().sum().sqrt()
    coef = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0).float()
    rate = (s["lr"] / (1 - b1 ** t)).float()
    root = (1 / torch.sqrt(1 - b2 ** t)).float()
    g = s["g"].float() * coef
    if s["bits"] == 32:
        m, v = s["m"], s["v"]
    else:
        m = s["m"].view(-1, BLOCK).float() * s["ms"][:, None]
        r = s["v"].view(-1, BLOCK).float() * s["vs"][:, None]
        m, v = m.view(-1), (r * r).view(-1)
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * g * (1 - b2)
    r = v.sqrt()
    p = s["p"] * (1 - s["lr"] * DECAY) - rate * (m / (r * root + EPS))
    s["p"].copy_(p)
    if s["shadow"] is not None:
        s["shadow"].copy_(p)
    if s["bits"] == 32:
        s["m"].copy_(m)
        s["v"].copy_(v)
    else:
        m, r = m.view(-1, BLOCK), r.view(-1, BLOCK)
        codes, scale = _quantise(m, m.abs().amax(1))
        s["m"].copy_(codes.view(-1))
        s["ms"].copy_(scale)
        codes, scale = _quantise_root(r, s["place"], s["step"])
        s["v"].copy_(codes.view(-1))
        s["vs"].copy_(scale)
    return _adamw_out(s, norm.float())


def _adamw_out(s, norm):
    return {"p": s["p"], "m": s["m"], "v": s["v"], "m_scale": s["ms"],
            "v_scale": s["vs"], "shadow": s["shadow"], "step": s["step"],
            "norm": norm.reshape(1)}


def run(state):
    s = state
    if not own:
        if s["op"] == "adamw":
            return _plain_adamw(s)
        if s["op"] == "step":
            return _plain_step(s)
        return _plain_recurrence(s, s["op"] == "train")

    if s["op"] == "adamw":
        from zaremba_amd.ops.adamw import adamw_step_
        x = s["lists"]
        norm = adamw_step_(x["p"], x["g"], x["m"], x["v"], s["step"],
                           lr=s["lr"], betas=BETAS, eps=EPS,
                           weight_decay=DECAY, max_norm=s["max_norm"],
                           exp_avg_scales=x["ms"], exp_avg_sq_scales=x["vs"],
                           shadows=x["shadow"])
        return _adamw_out(s, norm)
    from zaremba_amd.ops import glr
    if s["op"] == "step":
        return {"h": glr.glr_step(s["gates"], s["c0"]), "c": s["c0"]}
    if s["op"] == "forward":
        h, cT, _ = glr.glr_forward(s["gates"], s["c0"], s["lengths"])
        return {"h": h, "cT": cT}
    h, cT, marks = glr.glr_forward(s["gates"], s["c0"], s["lengths"],
                                   training=True)
    dgates, dc0 = glr.glr_backward(s["dh"], s["dcT"], s["gates"], s["c0"],
                                   marks, s["lengths"])
    return {"h": h, "cT": cT, "dgates": dgates, "dc0": dc0}


# ---------------------------------------------------------------------------
# the definitions in 64 bits, step by step
# ---------------------------------------------------------------------------

def _exact_recurrence(case, s):
    gates = s["gates"].double()
    if case["op"] == "step":
        gates = gates[None]
    T, B, H = gates.size(0), gates.size(1), gates.size(2) // 4
    squash = lambda x: 1 / (1 + torch.exp(-x))  # noqa: E731
    i, f, o = (squash(gates[..., k * H:(k + 1) * H]) for k in range(3))
    n = torch.tanh(gates[..., 3 * H:])
    del gates
    lengths = s["lengths"]
    if lengths is not None:
        ends = lengths.tolist()
        dead = torch.ones(T, B, 1, dtype=torch.bool, device=DEVICE)
        for b in range(B):
            dead[:ends[b], b] = False
        f.masked_fill_(dead, 1.0)
        i.masked_fill_(dead, 0.0)
        o.masked_fill_(dead, 0.0)
    b = i * n
    c = torch.empty(T + 1, B, H, dtype=torch.float64, device=DEVICE)
    c[0] = s["c0"]
    for t in range(T):
        torch.addcmul(b[t], f[t], c[t], out=c[t + 1])
    h = torch.tanh(c[1:]).mul_(o)
    if case["op"] == "step":
        return {"h": h[0], "c": c[1]}
    out = {"h": h, "cT": c[T].clone()}
    if case["op"] == "forward":
        return out
    del b
    tc = torch.tanh(c[1:])
    dh = s["dh"].double()
    g = dh * o * (1 - tc ** 2)
    carry = s["dcT"].double()
    for t in range(T - 1, -1, -1):
        g[t] += carry
        carry = f[t] * g[t]
    out["dc0"] = carry
    d = torch.empty(T, B, 4 * H, dtype=torch.float64, device=DEVICE)
    d[..., 2 * H:3 * H] = dh.mul_(tc).mul_(o).mul_(1 - o)
    del tc, dh
    d[..., :H] = g * n * i * (1 - i)
    d[..., H:2 * H] = g * c[:T] * f * (1 - f)
    d[..., 3 * H:] = g * i * (1 - n ** 2)
    if lengths is not None:
        d.masked_fill_(dead, 0.0)
    out["dgates"] = d
    return out


def _exact_adamw(case, s):
    b1, b2 = BETAS
    t = int(s["step"]) + 1
    g = s["g"].double()
    norm = torch.linalg.vector_norm(g)
    g *= min(1.0, s["max_norm"] / (float(norm) + 1e-6))
    if case["bits"] == 32:
        m, v = s["m"].double(), s["v"].double()
    else:
        m = s["m"].double().view(-1, BLOCK) * s["ms"].double()[:, None]
        v = (s["v"].double().view(-1, BLOCK)
             * s["vs"].double()[:, None]) ** 2
        m, v = m.view(-1), v.view(-1)
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g ** 2
    del g
    step = m / (1 - b1 ** t) / (torch.sqrt(v / (1 - b2 ** t)) + EPS)
    p = s["p"].double() * (1 - s["lr"] * DECAY) - s["lr"] * step
    out = {"p": p, "step": s["step"] + 1, "norm": norm.reshape(1),
           "shadow": p if case["shadow"] else None}
    if case["bits"] == 32:
        return dict(out, m=m, v=v, m_scale=None, v_scale=None)
    for k, x in (("m", m.view(-1, BLOCK)), ("v", v.sqrt().view(-1, BLOCK))):
        scale = x.abs().max(1).values / E4M3_MAX
        scale[scale < TINY / E4M3_MAX] = 0
        out[k + "_scale"] = scale
        out[k] = torch.where(scale[:, None] > 0, x / scale[:, None],
                             torch.zeros_like(x)).view(-1)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "adamw":
        return _exact_adamw(case, s)
    return _exact_recurrence(case, s)
