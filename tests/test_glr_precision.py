"""The gated linear recurrence in float32, value by value.

A running error analysis in 64 bits gives each output a bound of its own, so
that a small gradient beside a large one has to be right in its own digits.
With u = 2^-24, half a step of float32, and hardware exponentials and
reciprocals that are off by one whole step (2 u):

  s(x) = 1 / (1 + exp(-x)): the exponent is rounded and so is its factor
    log2 e, 2 |x| u of exp(-x), and 2 u of the exponential; the sum u, the
    reciprocal 2 u. Together SIG(x) = (5 + 2 |x|) u of the value.
  tanh: 16 u of the value (csrc/glr.hip: a series under 1/8; from there
    exp(-2|x|) is off by (4 |x| + 2) u, which 1 - exp(-2|x|) sees as at most
    12 u at 1/8 and less above; the quotient 4 u). With gates in 16 bits x
    itself stands for its tanh under 2^-8, off by x^2 / 3 < 86 u, and at 2^-8
    the same formula is off by 2.5 u / 0.0078 + 4 u: 330 u.
  c_t = f_t c_{t-1} + y_t, y = s(i) tanh(n): each product and sum is rounded,
    and so is the product of the f's by which steps are composed: 3 u of a
    state's part at each step, 4 u of the sum of the magnitudes that c_t is
    made of (C below) for the sums at the three levels of composition.

What follows adds these up through the formulas. The products of two errors
are covered by one hundredth more.
"""

import pytest
import torch

from zaremba_amd.ops import glr as G

GPU = pytest.mark.gpu
U = 2.0 ** -24


def tanh_error(dtype):
    return (330 if torch.finfo(dtype).bits == 16 else 16) * U


def sig(x):
    return (5 + 2 * x.abs()) * U


def bounds(gates, c0, dh, dcT):
    """(value, bound) of h, cT, dgates and dc0, in 64 bits from the formulas,
    for outputs that are not rounded further."""
    TANH = tanh_error(gates.dtype)
    gates, c0, dh, dcT = (x.detach().double().cpu()
                          for x in (gates, c0, dh, dcT))
    T = gates.size(0)
    xi, xf, xo, xn = gates.chunk(4, -1)
    i, f, o, n = xi.sigmoid(), xf.sigmoid(), xo.sigmoid(), xn.tanh()
    # 1 - s(x) and 1 - tanh(x)^2 without cancellation
    i1, f1, o1 = (-xi).sigmoid(), (-xf).sigmoid(), (-xo).sigmoid()
    slope = lambda x: 1 / torch.cosh(x) ** 2  # noqa: E731
    c, C, E = [c0], [c0.abs()], [torch.zeros_like(c0)]
    for t in range(T):
        y = i[t] * n[t]
        c.append(f[t] * c[-1] + y)
        C.append(f[t] * C[-1] + y.abs())
        E.append(f[t] * E[-1] + f[t] * C[-2] * (sig(xf[t]) + 3 * U)
                 + y.abs() * (TANH + sig(xi[t]) + 2 * U) + 4 * U * C[-1])
    before, after = torch.stack(c[:-1]), torch.stack(c[1:])
    Eb, Ea = torch.stack(E[:-1]), torch.stack(E[1:])
    tc, sl = after.tanh(), slope(after)
    Et = (sl + 2 * Ea) * Ea + TANH * tc.abs()
    h = o * tc
    eh = o * Et + h.abs() * (sig(xo) + 3 * U)
    u = dh * o * sl
    eu = (dh * o).abs() * (2 * tc.abs() * Et + 2 * U
                           + (sig(xo) + 2 * U) * sl)
    g, S, Eg = [None] * T, [None] * T, [None] * T
    carry, size, err = dcT, dcT.abs(), torch.zeros_like(dcT)
    for t in range(T - 1, -1, -1):
        g[t], S[t] = u[t] + carry, u[t].abs() + size
        Eg[t] = err + eu[t] + 4 * U * S[t]
        carry, size = f[t] * g[t], f[t] * S[t]
        err = f[t] * Eg[t] + size * (sig(xf[t]) + 3 * U)
    g, Eg = torch.stack(g), torch.stack(Eg)
    part = lambda s, x: (sig(x) + 4 * U) * (1 - s) + s * sig(x) + U  # noqa
    rows = [
        (g * n * i * i1, Eg * (n * i * i1).abs()
         + (g * n * i).abs() * (part(i, xi) + TANH * i1)),
        (g * before * f * f1, (Eg * before.abs() + (g * Eb).abs()) * f * f1
         + (g * before * f).abs() * part(f, xf)),
        (dh * tc * o * o1, dh.abs() * o * o1 * Et
         + (dh * tc * o).abs() * part(o, xo)),
        (g * i * slope(xn), Eg * i * slope(xn) + (g * i).abs()
         * ((sig(xi) + 4 * U) * slope(xn) + 2 * n ** 2 * TANH + 2 * U))]
    d, ed = (torch.cat([r[k] for r in rows], -1) for k in (0, 1))
    return {"h": (h, eh), "cT": (c[-1], E[-1]), "dgates": (d, ed),
            "dc0": (carry, err)}


def outside(got, want, bound):
    """How many values of `got` are not `want`, within `bound` and one
    rounding to the type of `got`."""
    info = torch.finfo(got.dtype)
    got = got.double().cpu()
    half = want.abs() * info.eps / 2 if info.bits < 32 else 0.0
    allowed = 1.01 * bound + half + info.tiny * info.eps
    return int((~((got - want).abs() <= allowed)).sum())


def make(T, B, H, device="cpu", dtype=torch.float32, small=1.0, seed=0):
    """Gates of 1.5; what enters and the first state are `small` of that."""
    gen = torch.Generator().manual_seed(seed)
    gates = torch.randn(T, B, 4 * H, generator=gen) * 1.5
    gates[..., 3 * H:] *= small
    c0 = torch.randn(B, H, generator=gen) * small
    dh = torch.randn(T, B, H, generator=gen).to(dtype)
    dcT = torch.randn(B, H, generator=gen)
    return [x.to(device) for x in (gates.to(dtype), c0, dh, dcT)]


def outputs(gates, c0, dh, dcT):
    h, cT, marks = G.glr_forward(gates, c0, training=True)
    dgates, dc0 = G.glr_backward(dh, dcT, gates, c0, marks)
    return {"h": h, "cT": cT, "dgates": dgates, "dc0": dc0}


def check(x):
    got, want = outputs(*x), bounds(*x)
    for name, (value, bound) in want.items():
        assert outside(got[name], value, bound) == 0, name


SMALL = [1.0, 1e-2, 1e-3, 1e-4, 1e-5, 1e-7]


@pytest.mark.parametrize("small", SMALL)
def test_eager_within_its_roundings(small):
    for size in ((1, 3, 5), (35, 4, 40), (200, 2, 9)):
        check(make(*size, small=small))


def test_the_bounds_are_narrow():
    """Mistakes planted in the 64-bit values are seen: 0.1 %, 11 bits, a
    dropped gradient, and a tanh that holds 24 bits of 1 only."""
    x = make(35, 20, 65)
    want = bounds(*x)
    d, bound = want["dgates"]
    many = d.numel()
    assert outside(d.float(), d, bound) == 0
    assert outside((d * 1.001).float(), d, bound) > 0.95 * many
    assert outside(d.half().float(), d, bound) > 0.8 * many
    assert outside(torch.zeros_like(d, dtype=torch.float32), d,
                   bound) > 0.99 * many
    for small in (1e-3, 1e-5, 1e-7):
        x = make(1, 20, 65, small=small)
        h, bound = bounds(*x)["h"]
        o = x[0].double().chunk(4, -1)[2].sigmoid()
        coarse = torch.round(h / o / U) * U * o
        assert outside(coarse.float(), h, bound) > 0.5 * h.numel(), small


def test_the_values_are_the_gradients():
    """The closed forms above against autograd in 64 bits."""
    gates, c0, dh, dcT = (x.double() for x in make(9, 3, 4))
    gates, c0 = gates.requires_grad_(), c0.requires_grad_()
    h, cT = G.glr(gates, c0)
    dg, dc0 = torch.autograd.grad((h * dh).sum() + (cT * dcT).sum(),
                                  (gates, c0))
    want = bounds(gates, c0, dh, dcT)
    for got, name in ((h, "h"), (cT, "cT"), (dg, "dgates"), (dc0, "dc0")):
        # some hundred roundings of 2^-53 of numbers of a few units
        assert float((got.detach() - want[name][0]).abs().max()) < 1e-13


@GPU
@pytest.mark.parametrize("small", SMALL)
def test_kernels_within_their_roundings(small):
    """Windows of one tile, chains in either kind of tile, and odd sizes."""
    for size in ((1, 3, 5), (35, 20, 650), (64, 3, 70), (128, 2, 33),
                 (129, 17, 1001), (700, 3, 40), (5000, 1, 72)):
        check(make(*size, device="cuda", small=small))


@GPU
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("small", [1.0, 1e-4, 1e-6])
def test_kernels_in_16_bits_add_one_rounding(dtype, small):
    for size in ((35, 20, 200), (300, 3, 70)):
        check(make(*size, device="cuda", dtype=dtype, small=small))


@GPU
@pytest.mark.parametrize("small", SMALL)
def test_steps_within_their_roundings(small):
    gates, c0, dh, dcT = make(3, 20, 201, device="cuda", small=small)
    want = bounds(gates, c0, dh, dcT)
    c = c0.clone()
    for t in range(3):
        h = G.glr_step(gates[t], c)
        value, bound = want["h"]
        assert outside(h, value[t], bound[t]) == 0, t
    assert outside(c, *want["cT"]) == 0


@GPU
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16,
                                   torch.float16])
@pytest.mark.parametrize("T,B,H", [(35, 6, 40), (128, 5, 9), (700, 6, 70)])
def test_padded_rows_within_their_roundings(dtype, T, B, H):
    """Each row of a padded batch, batch first, as the window that it is."""
    gen = torch.Generator().manual_seed(1)
    gates, c0, dh, dcT = make(T, B, H, "cuda", dtype)
    first = lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)  # noqa
    gates, dh = first(gates), first(dh)
    ends = torch.randint(1, T + 1, (B,), generator=gen).tolist()
    ends[0], ends[-1] = 0, T
    for b, n in enumerate(ends):
        gates[n:, b], dh[n:, b] = float("nan"), float("inf")
    lengths = torch.tensor(ends, device="cuda")
    h, cT, marks = G.glr_forward(gates, c0, lengths, training=True)
    dgates, dc0 = G.glr_backward(dh, dcT, gates, c0, marks, lengths)
    for b, n in enumerate(ends):
        row = slice(b, b + 1)
        assert not h[n:, b].any() and not dgates[n:, b].any()
        if n == 0:
            assert torch.equal(cT[b], c0[b]) and torch.equal(dc0[b], dcT[b])
            continue
        want = bounds(gates[:n, row], c0[row], dh[:n, row], dcT[row])
        for name, got in (("h", h[:n, row]), ("cT", cT[row]),
                          ("dgates", dgates[:n, row]), ("dc0", dc0[row])):
            assert outside(got, *want[name]) == 0, (name, b)
