"""The gated linear recurrence against a plain implementation in 64 bits.

Tolerances. An output in type t is the 64-bit value rounded once, off by at
most finfo(t).eps / 2 of the value, plus the error of the 32-bit state before
it. A step's factors (products of a sigmoid and a tanh, each from one
exponential and one reciprocal) are off by a few units of 2^-24 of numbers of
at most 1, so a state of size C is off by at most about 16 * 2^-24 * (1 + C)
at each step, and errors older than a step shrink by its forget gate: with
sigmoid(f) <= F the sum is under 16 * 2^-24 * (1 + C) / (1 - F). The gates
drawn below keep F <= 0.95 in the mean over a step's neighbours, which
gives 2^-24 * 320 * (1 + C); an h or a gate gradient is a product of these with
factors of at most 1 and the upstream gradient.
"""

import pytest
import torch

from zaremba_amd.ops import glr as G
from zaremba_amd.ops import functional as F_ref

GPU = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
STATE = 320 * 2.0 ** -24


def make(T, B, H, dtype, device, batch_first=False, ragged=False, seed=0,
         scale=1.5):
    gen = torch.Generator().manual_seed(seed)
    shape = (B, T) if batch_first else (T, B)
    gates = (torch.randn(*shape, 4 * H, generator=gen) * scale).to(dtype)
    dh = torch.randn(*shape, H, generator=gen).to(dtype)
    gates, dh = gates.to(device), dh.to(device)
    if batch_first:
        gates, dh = gates.transpose(0, 1), dh.transpose(0, 1)
    c0 = torch.randn(B, H, generator=gen).to(device)
    dcT = torch.randn(B, H, generator=gen).to(device)
    lengths = None
    if ragged:
        lengths = torch.randint(0, T + 1, (B,), generator=gen)
        lengths[0] = 0
        lengths[-1] = T
        lengths = lengths.to(device)
    return gates, c0, dh, dcT, lengths


def oracle(gates, c0, dh, dcT, lengths):
    """h, cT, dgates, dc0 in 64 bits on the CPU, from the formulas."""
    g = gates.detach().double().cpu()
    T, B, H = g.size(0), g.size(1), g.size(2) // 4
    dh = torch.zeros(T, B, H) if dh is None else dh
    dh = dh.detach().double().cpu()
    z = torch.zeros(B, H, dtype=torch.float64)
    c = z if c0 is None else c0.detach().double().cpu()
    live = torch.ones(T, B, 1, dtype=torch.bool)
    if lengths is not None:
        live = (torch.arange(T)[:, None] < lengths.cpu()[None])[..., None]
    g = torch.where(live, g, torch.zeros_like(g))
    dh = torch.where(live, dh, torch.zeros_like(dh))
    i, f, o = (torch.sigmoid(g[..., k * H:(k + 1) * H]) for k in range(3))
    n = torch.tanh(g[..., 3 * H:])
    states = [c]
    for t in range(T):
        new = f[t] * c + i[t] * n[t]
        c = torch.where(live[t], new, c)
        states.append(c)
    cs = torch.stack(states)
    tc = torch.tanh(cs[1:])
    h = torch.where(live, o * tc, torch.zeros_like(tc))
    carry = z if dcT is None else dcT.detach().double().cpu()
    d = torch.zeros(T, B, 4 * H, dtype=torch.float64)
    for t in range(T - 1, -1, -1):
        dc = carry + dh[t] * o[t] * (1 - tc[t] ** 2)
        row = torch.cat([dc * n[t] * i[t] * (1 - i[t]),
                         dc * cs[t] * f[t] * (1 - f[t]),
                         dh[t] * tc[t] * o[t] * (1 - o[t]),
                         dc * i[t] * (1 - n[t] ** 2)], 1)
        d[t] = torch.where(live[t], row, torch.zeros_like(row))
        carry = torch.where(live[t], f[t] * dc, carry)
    return h, c, d, carry, cs


def near(got, want, size, name):
    """got is want rounded to its type, `size`: the error scale of want."""
    assert got.shape == want.shape, name
    half = torch.finfo(got.dtype).eps / 2
    least = torch.finfo(got.dtype).tiny
    want = want.to(got.device)
    off = (got.double() - want).abs()
    allowed = want.abs() * half + size * STATE * (1 + half) + least
    assert bool((off <= allowed).all()), (
        name, float((off - allowed).max()), float(off.max()))


def check(gates, c0, dh, dcT, lengths):
    h, cT, marks = G.glr_forward(gates, c0, lengths, training=True)
    dgates, dc0 = G.glr_backward(dh, dcT, gates, c0, marks, lengths)
    wh, wc, wd, wdc0, cs = oracle(gates, c0, dh, dcT, lengths)
    size = 1 + float(cs.abs().max()) if cs.numel() else 1.0
    up = 1.0
    if dh is not None and dh.numel():
        live = torch.ones_like(dh[..., :1], dtype=torch.bool)
        if lengths is not None:
            live = (torch.arange(dh.size(0), device=dh.device)[:, None]
                    < lengths[None])[..., None]
        up += float(torch.where(live, dh, torch.zeros_like(dh)).float()
                    .abs().max())
    if dcT is not None and dcT.numel():
        up += float(dcT.abs().max())
    assert h.dtype == gates.dtype and dgates.dtype == gates.dtype
    assert cT.dtype == torch.float32 and dc0.dtype == torch.float32
    near(h, wh, size, "h")
    near(cT, wc, size, "cT")
    # the carried gradient adds up over 1 / (1 - F) steps as the state does
    near(dgates, wd, size * up * 4, "dgates")
    near(dc0, wdc0, size * up * 4, "dc0")
    return h, cT, dgates, dc0


def cases(device):
    dev = torch.device(device)
    for T, B, H in [(1, 1, 1), (1, 3, 5), (2, 1, 64), (7, 2, 130),
                    (35, 20, 12), (63, 1, 3), (64, 2, 4), (65, 3, 8),
                    (130, 2, 33)]:
        yield T, B, H, dev


@pytest.mark.parametrize("ragged", [False, True])
def test_eager_matches_oracle(ragged):
    for T, B, H, dev in cases("cpu"):
        check(*make(T, B, H, torch.float32, dev, ragged=ragged))


def test_eager_gradcheck():
    gates, c0, _, _, lengths = make(5, 3, 2, torch.float64, "cpu",
                                    ragged=True)
    gates, c0 = gates.requires_grad_(), c0.double().requires_grad_()
    assert torch.autograd.gradcheck(
        lambda g, c: G.glr(g, c, lengths), (gates, c0))


def test_oracle_against_differences():
    """The oracle's gradient against central differences of its loss."""
    gates, c0, dh, dcT, lengths = make(6, 3, 2, torch.float64, "cpu",
                                       ragged=True)
    c0, dcT = c0.double(), dcT.double()

    def loss(g, c):
        h, cT = oracle(g, c, None, None, lengths)[:2]
        return (h * dh).sum() + (cT * dcT).sum()

    _, _, d, dc0, _ = oracle(gates, c0, dh, dcT, lengths)
    eps = 1e-6
    for x, grad in ((gates, d), (c0, dc0)):
        flat, at = x.view(-1), grad.reshape(-1)
        for k in range(0, flat.numel(), 3):
            keep = float(flat[k])
            flat[k] = keep + eps
            up = loss(gates, c0)
            flat[k] = keep - eps
            down = loss(gates, c0)
            flat[k] = keep
            # the difference is off by eps^2 and by 1e-16 * |loss| / eps
            assert abs(float(up - down) / (2 * eps) - float(at[k])) < 1e-8


def refusals(device):
    gates, c0, dh, dcT, _ = make(4, 3, 2, torch.float32, device)
    bad = [
        lambda: G.glr_forward(gates[0], c0),
        lambda: G.glr_forward(gates[..., :7], c0),
        lambda: G.glr_forward(gates.int(), c0),
        lambda: G.glr_forward(gates, c0[:2]),
        lambda: G.glr_forward(gates, c0.half()),
        lambda: G.glr_forward(gates, c0, torch.tensor([1., 2., 3.],
                                                      device=device)),
        lambda: G.glr_forward(gates, c0, torch.tensor([1, 2],
                                                      device=device)),
        lambda: G.glr_step(gates, c0),
        lambda: G.glr_step(gates[0], c0[:, :1]),
        lambda: G.glr_step(gates[0].clone().requires_grad_(), c0),
        lambda: G.glr_backward(dh, dcT[:1], gates, c0, None),
    ]
    return bad


def test_refusals_eager():
    for call in refusals("cpu"):
        with pytest.raises(RuntimeError, match="glr"):
            call()


def test_refusals_eager_of_outputs_and_gradients():
    """Those of the kernels: nothing is spread over a larger `out`, and no
    type is changed on the way."""
    gates, c0, dh, dcT, _ = make(4, 3, 2, torch.float32, "cpu")
    for call in (
            lambda: G.glr_forward(gates, c0, out=torch.zeros(5, 4, 3, 2)),
            lambda: G.glr_forward(gates, c0, out=torch.zeros(4, 3, 3)),
            lambda: G.glr_forward(gates, c0, out=dh.half()),
            lambda: G.glr_backward(dh, dcT, gates, c0, None,
                                   out=torch.zeros(2, 4, 3, 8)),
            lambda: G.glr_backward(dh, dcT, gates, c0, None,
                                   out=gates.double()),
            lambda: G.glr_backward(dh.half(), dcT, gates, c0, None),
            lambda: G.glr_backward(dh[:2], dcT, gates, c0, None)):
        with pytest.raises(RuntimeError, match="glr"):
            call()
    h, d = torch.zeros_like(dh), torch.zeros_like(gates)
    assert G.glr_forward(gates, c0, out=h)[0] is h
    assert G.glr_backward(dh, dcT, gates, c0, None, out=d)[0] is d
    assert h.any() and d.any()


def test_no_steps_and_no_rows_eager():
    for T, B, H in [(0, 3, 4), (5, 0, 4), (5, 3, 0), (0, 0, 0)]:
        gates, c0, dh, dcT, _ = make(T, B, H, torch.float32, "cpu")
        h, cT, dgates, dc0 = check(gates, c0, dh, dcT, None)
        assert h.shape == (T, B, H) and dgates.shape == gates.shape
        d, dc0 = G.glr_backward(None, None, gates, None, None)
        assert d.shape == gates.shape and not dc0.any()
        c = c0.clone().requires_grad_()
        h, cT = G.glr(gates, c)
        (cT * dcT).sum().backward()
        assert c.grad.shape == c0.shape


def test_step_is_the_scan_eager():
    gates, c0, *_ = make(9, 4, 6, torch.float32, "cpu")
    h, cT, _ = G.glr_forward(gates, c0)
    c = c0.clone()
    for t in range(9):
        assert torch.equal(G.glr_step(gates[t], c), h[t])
    assert torch.equal(c, cT)


# ---------------------------------------------------------------------------
# kernels
# ---------------------------------------------------------------------------

@GPU
def test_refusals_gpu():
    for call in refusals("cuda"):
        with pytest.raises(RuntimeError, match="glr"):
            call()
    gates, c0, dh, dcT, _ = make(4, 3, 2, torch.float32, "cuda")
    _, _, marks = G.glr_forward(gates, c0, training=True)
    for call in (
            lambda: G.glr_forward(gates.double(), c0),
            lambda: G.glr_forward(gates, c0.cpu()),
            lambda: G.glr_forward(gates, c0, torch.tensor([1, 2, 3])),
            lambda: G.glr_forward(gates, c0, out=gates[..., :2]),
            lambda: G.glr_forward(gates, c0, out=gates.view(-1)[:24].view(
                4, 3, 2)),
            lambda: G.glr_backward(dh, dcT, gates, c0, marks, out=gates),
            lambda: G.glr_backward(dh, dcT, gates, c0, marks,
                                   out=gates[:3].clone()),
            lambda: G.glr_step(gates[0], gates.view(-1)[:6].view(3, 2)),
            lambda: G.glr_backward(dh.half(), dcT, gates, c0, marks),
            lambda: G.glr_backward(dh[:2], dcT, gates, c0, marks),
            lambda: G.glr_backward(dh, dcT, gates, c0, marks[..., :1]),
            lambda: G.glr_backward(dh, dcT, gates, c0, marks.double()),
            lambda: G.glr_step(gates[0], c0[:1].expand(3, 2)),
            lambda: G.glr_step(gates[0], c0.double())):
        with pytest.raises(RuntimeError, match="glr"):
            call()


@GPU
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("batch_first", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_kernels_match_oracle(dtype, batch_first, ragged):
    for T, B, H, dev in cases("cuda"):
        check(*make(T, B, H, dtype, dev, batch_first, ragged))


@GPU
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,B,H", [(35, 20, 1500), (35, 20, 650),
                                   (257, 5, 1001), (4099, 1, 72),
                                   (20000, 2, 12), (1030, 64, 40)])
def test_kernels_match_oracle_larger(T, B, H, dtype):
    check(*make(T, B, H, dtype, "cuda", ragged=B > 1))


@GPU
def test_without_states_and_with_one_gradient():
    gates, c0, dh, dcT, lengths = make(70, 3, 17, torch.float32, "cuda",
                                       ragged=True)
    check(gates, None, dh, dcT, lengths)
    check(gates, c0, None, dcT, lengths)
    check(gates, c0, dh, None, lengths)
    check(gates, None, dh, None, lengths.int())


@GPU
def test_no_steps_and_no_rows():
    for T, B, H in [(0, 3, 4), (5, 0, 4), (5, 3, 0)]:
        gates, c0, dh, dcT, _ = make(T, B, H, torch.bfloat16, "cuda")
        h, cT, dgates, dc0 = check(gates, c0, dh, dcT, None)
        assert h.shape == (T, B, H) and dgates.shape == gates.shape
    assert G.glr_step(torch.empty(0, 8, device="cuda"),
                      torch.empty(0, 2, device="cuda")).shape == (0, 2)


@GPU
@pytest.mark.parametrize("dtype", TYPES)
def test_padding_has_no_effect(dtype):
    """Lengths beyond both ends, all rows empty, and NaN in the padding."""
    gates, c0, dh, dcT, _ = make(71, 4, 37, dtype, "cuda")
    lengths = torch.tensor([-5, 71, 1000, 40], device="cuda")
    clean = check(gates, c0, dh, dcT, lengths.clamp(0, 71))
    live = (torch.arange(71, device="cuda")[:, None]
            < lengths[None])[..., None]
    nan = torch.full_like(gates, float("nan"))
    gates = torch.where(live, gates, nan)
    dh = torch.where(live, dh, nan[..., :37])
    h, cT, marks = G.glr_forward(gates, c0, lengths, training=True)
    dgates, dc0 = G.glr_backward(dh, dcT, gates, c0, marks, lengths)
    for got, want in zip((h, cT, dgates, dc0), clean):
        assert torch.equal(got, want)
    none = torch.zeros(4, dtype=torch.int32, device="cuda")
    h, cT, marks = G.glr_forward(gates, c0, none, training=True)
    dgates, dc0 = G.glr_backward(dh, dcT, gates, c0, marks, none)
    assert not h.any() and not dgates.any()
    assert torch.equal(cT, c0) and torch.equal(dc0, dcT)


@GPU
@pytest.mark.parametrize("dtype", TYPES)
def test_closed_and_open_gates(dtype):
    """Gates at both infinities and at the type's ends: a closed forget gate
    drops the state exactly, an open one keeps it exactly."""
    inf = float("inf")
    T, B, H = 66, 2, 5
    gates, c0, dh, dcT, _ = make(T, B, H, dtype, "cuda")
    low = torch.finfo(dtype).min
    for shut, wide in ((-inf, inf), (low, -low)):
        g = gates.clone()
        g[..., :H] = shut                 # nothing enters
        g[..., H:2 * H] = wide            # everything stays
        h, cT, marks = G.glr_forward(g, c0, training=True)
        assert torch.equal(cT, c0)
        dgates, dc0 = G.glr_backward(dh, dcT, g, c0, marks)
        assert bool(torch.isfinite(dgates).all())
        assert not dgates[..., :2 * H].any()
        g[40, :, H:2 * H] = shut          # and is dropped at step 40
        h, cT, marks = G.glr_forward(g, c0, training=True)
        assert not cT.any() and not h[40:].any()
        dgates, dc0 = G.glr_backward(dh, dcT, g, c0, marks)
        assert bool(torch.isfinite(dgates).all())


@GPU
@pytest.mark.parametrize("T", [70, 700])
def test_nan_stays_in_its_channel(T):
    """In one tile, and through a chain, forward and backward."""
    gates, c0, dh, dcT, _ = make(T, 3, 9, torch.float32, "cuda")
    gates[30, 1, 4] = float("nan")
    h, cT, marks = G.glr_forward(gates, c0, training=True)
    bad = torch.isnan(h)
    assert bool(bad[30:, 1, 4].all()) and int(bad.sum()) == T - 30
    assert int(torch.isnan(cT).sum()) == 1
    dh[20, 0, 7] = float("nan")
    d, dc0 = G.glr_backward(dh, dcT, gates, c0, marks)
    bad = torch.isnan(d.view(T, 3, 4, 9)).any(2)
    assert bool(bad[:, 1, 4].all())          # NaN states give NaN gradients
    assert bool(bad[:21, 0, 7].all()) and int(bad[:, 0, 7].sum()) == 21
    assert int(bad.sum()) == T + 21
    assert int(torch.isnan(dc0).sum()) == 2


@GPU
def test_writes_are_seen_by_autograd():
    """A tensor that a graph has saved and a kernel then overwrites."""
    gates, c0, *_ = make(4, 3, 2, torch.float32, "cuda")
    w = torch.ones(3, 2, device="cuda", requires_grad=True)
    c = c0.clone()
    y = (w * c).sum()
    with torch.no_grad():
        G.glr_step(gates[0], c)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()


@GPU
@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_alignment(dtype):
    """Sliced, offset, expanded and unevenly strided inputs."""
    T, B, H = 37, 3, 24
    wide, c0, dh, dcT, _ = make(T + 2, B + 1, H + 3, dtype, "cuda")
    gates = wide[1:T + 1, 1:, 5:5 + 4 * H]
    dh = dh[1:T + 1, :B, 1:1 + H]
    assert not gates.is_contiguous()
    check(gates, c0[:B, 2:2 + H], dh, dcT[1:, 1:1 + H], None)
    check(wide[::2, ::2, :4 * H][:18, :2], c0[:2, :H], dh[:18, :2],
          dcT[:2, :H], None)
    one = gates[:, :1].expand(T, B, 4 * H)
    check(one, c0[:1, :H].expand(B, H), dh[:1].expand(T, B, H),
          dcT[:B, :H], None)
    skipped = wide[:T, :B, ::1].flip(2)[..., :4 * H]  # a copy
    check(skipped, c0[:B, :H], dh, dcT[:B, :H], None)
    every = wide[:T, :B, ::2][..., :4 * (H // 4)]     # the last axis apart
    check(every, c0[:B, :H // 4], dh[..., ::4], dcT[:B, :H // 4], None)


@GPU
def test_out_is_written_and_nothing_behind():
    gates, c0, dh, dcT, lengths = make(40, 3, 21, torch.bfloat16, "cuda",
                                       ragged=True)
    n, m = 40 * 3 * 21, 40 * 3 * 84
    room = torch.full((2, m + 64), 7.0, dtype=torch.bfloat16, device="cuda")
    h = room[0, :n].view(40, 3, 21)
    d = room[1, :m].view(40, 3, 84)
    h1, _, marks = G.glr_forward(gates, c0, lengths, training=True, out=h)
    d1, _ = G.glr_backward(dh, dcT, gates, c0, marks, lengths, out=d)
    assert h1.data_ptr() == h.data_ptr() and d1.data_ptr() == d.data_ptr()
    h2, _, marks = G.glr_forward(gates, c0, lengths, training=True)
    d2, _ = G.glr_backward(dh, dcT, gates, c0, marks, lengths)
    assert torch.equal(h, h2) and torch.equal(d, d2)
    assert bool((room[0, n:] == 7).all()) and bool((room[1, m:] == 7).all())


@GPU
def test_autograd_of_broadcast_and_shared_inputs():
    gates, c0, dh, dcT, lengths = make(38, 4, 10, torch.float32, "cuda",
                                       ragged=True)
    bias = torch.zeros(40, device="cuda", requires_grad=True)
    start = c0[:1].clone().requires_grad_()
    h, cT = G.glr(gates + bias, start.expand(4, 10), lengths)
    ((h * dh).sum() + (cT * dcT).sum()).backward()
    _, _, d, dc0, _ = oracle(gates, c0[:1].expand(4, 10), dh, dcT, lengths)
    near(bias.grad, d.sum((0, 1)), 38 * 4 * 16.0, "bias")
    near(start.grad, dc0.sum(0, keepdim=True), 4 * 16.0, "c0")
    # one gradient only, and none
    h, cT = G.glr(gates.clone().requires_grad_(), c0)
    cT.sum().backward()
    h, cT = G.glr(gates, c0)
    assert not h.requires_grad
    # the second derivative is refused
    x = gates.clone().requires_grad_()
    h, _ = G.glr(x, c0)
    (d,) = torch.autograd.grad(h.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()


@GPU
@pytest.mark.parametrize("dtype", TYPES)
def test_step_follows_the_scan(dtype):
    for B, H in [(1, 1), (20, 200), (3, 129), (64, 1500)]:
        gates, c0, *_ = make(6, B, H, dtype, "cuda")
        wh, wc, _, _, cs = oracle(gates, c0, None, None, None)
        pool = torch.full((B, H + 3), 5.0, device="cuda")
        c = pool[:, :H]
        c.copy_(c0)
        size = 1 + float(cs.abs().max())
        for t in range(6):
            near(G.glr_step(gates[t], c), wh[t], size, "h")
        near(c, wc, size, "c")
        assert bool((pool[:, H:] == 5).all())


@GPU
def test_same_bits_every_time():
    gates, c0, dh, dcT, lengths = make(500, 3, 130, torch.bfloat16, "cuda",
                                       ragged=True)
    a = G.glr_forward(gates, c0, lengths, training=True)
    b = G.glr_forward(gates, c0, lengths, training=True)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    a = G.glr_backward(dh, dcT, gates, c0, a[2], lengths)
    b = G.glr_backward(dh, dcT, gates, c0, b[2], lengths)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@GPU
@pytest.mark.parametrize("T,B,H", [(35, 4, 50), (3000, 1, 96)])
def test_captured_and_replayed(T, B, H):
    """Two graphs of the same call, replayed in turn with eager work between:
    each replay gives what the eager call gives for its inputs."""
    sets = [make(T, B, H, torch.bfloat16, "cuda", ragged=True, seed=s)
            for s in range(3)]
    def both(x):
        h, cT, marks = G.glr_forward(x[0], x[1], x[4], training=True)
        return (h, cT) + G.glr_backward(x[2], x[3], x[0], x[1], marks, x[4])

    want = [both(x) for x in sets]
    graphs = []
    for x in sets[:2]:
        at = [t.clone() for t in x]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            both(at)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = both(at)
        graphs.append((graph, at, got))
    for turn in range(4):
        for k, (graph, at, got) in enumerate(graphs):
            src = (turn + k) % 3
            for a, b in zip(at, sets[src]):
                a.copy_(b)
            graph.replay()
            both(sets[2])  # eager work beside it
            torch.cuda.synchronize()
            for a, b in zip(got, want[src]):
                assert torch.equal(a, b), (turn, k)


@GPU
def test_two_streams_at_once():
    sets = [make(2000, 1, 200, torch.bfloat16, "cuda", seed=s)
            for s in range(2)]
    want = [G.glr_forward(x[0], x[1], training=True) for x in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(5):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[k].append(G.glr_forward(sets[k][0], sets[k][1],
                                            training=True))
    torch.cuda.synchronize()
    for k in range(2):
        for r in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[k]))


@GPU
def test_offsets_past_32_bits():
    """A [T, B, 4H] view whose rows lie more than 2^31 elements apart."""
    T, B, H = 3, 2, 40
    apart = (1 << 30) + 8
    room = torch.empty(2 * apart + 2 * 160, dtype=torch.bfloat16,
                       device="cuda")
    gates = room.as_strided((T, B, 4 * H), (apart, 4 * H, 1))
    src, c0, dh, dcT, _ = make(T, B, H, torch.bfloat16, "cuda")
    gates.copy_(src)
    h, cT, marks = G.glr_forward(gates, c0, training=True)
    d, dc0 = G.glr_backward(dh, dcT, gates, c0, marks)
    h2, cT2, marks = G.glr_forward(src, c0, training=True)
    d2, dc02 = G.glr_backward(dh, dcT, src, c0, marks)
    assert torch.equal(h, h2) and torch.equal(d, d2)


@GPU
@pytest.mark.parametrize("T", [3, 400])
def test_rows_further_apart_than_an_offset_reaches(T):
    """Rows of the batch over 4 GB apart, in a loop and in a chain."""
    B, H = 3, 40
    apart = (1 << 31) + 24
    room = torch.empty(2 * apart + T * 4 * H, dtype=torch.bfloat16,
                       device="cuda")
    gates = room.as_strided((T, B, 4 * H), (4 * H, apart, 1))
    src, c0, dh, dcT, lengths = make(T, B, H, torch.bfloat16, "cuda",
                                     ragged=True)
    gates.copy_(src)
    h, cT, marks = G.glr_forward(gates, c0, lengths, training=True)
    d, dc0 = G.glr_backward(dh, dcT, gates, c0, marks, lengths)
    h2, cT2, marks2 = G.glr_forward(src, c0, lengths, training=True)
    d2, dc02 = G.glr_backward(dh, dcT, src, c0, marks2, lengths)
    for a, b in ((h, h2), (cT, cT2), (d, d2), (dc0, dc02)):
        near(a, b.double().cpu(), 16.0, "far rows")


@GPU
@pytest.mark.parametrize("T,B,H", [(40000, 1, 96), (3000, 9, 300)])
def test_same_bits_whatever_else_runs(T, B, H):
    """A long window is many blocks that wait for each other in an order that
    other work changes; its roundings are the same."""
    gates, c0, dh, dcT, _ = make(T, B, H, torch.float32, "cuda")
    load = torch.randn(1 << 24, device="cuda")
    side = torch.cuda.Stream()
    first = None
    for _ in range(12):
        with torch.cuda.stream(side):
            for _ in range(6):
                load.mul_(0.999)
        h, cT, marks = G.glr_forward(gates, c0, training=True)
        got = (h, cT, marks) + G.glr_backward(dh, dcT, gates, c0, marks)
        first = first or got
        assert all(torch.equal(x, y) for x, y in zip(got, first))
    torch.cuda.synchronize()


@GPU
@pytest.mark.parametrize("H", [9, 64, 70])
@pytest.mark.parametrize("ends", [
    [0, 1, 63, 64, 65, 127, 128, 129, 255, 256, 257, 383, 384, 385, 399, 400],
    [0] * 15 + [1], [128] * 16, [1, 400] * 8, [0] * 16])
def test_rows_that_end_at_tiles(H, ends):
    """Whole tiles of padding, with NaN there, and no step of some rows."""
    T, B = 400, len(ends)
    gates, c0, dh, dcT, _ = make(T, B, H, torch.bfloat16, "cuda")
    lengths = torch.tensor(ends, dtype=torch.int32, device="cuda")
    live = (torch.arange(T, device="cuda")[:, None]
            < lengths[None])[..., None]
    gates = gates.masked_fill(~live, float("nan"))
    dh = dh.masked_fill(~live, float("nan"))
    check(gates, c0, dh, dcT, lengths)


@GPU
def test_refusals_of_shared_memory_and_sizes():
    T, B, H = 8, 3, 4
    gates, c0, dh, dcT, _ = make(T, B, H, torch.float32, "cuda")
    _, _, marks = G.glr_forward(gates, c0, training=True)
    room = torch.zeros(T * B * 4 * H, device="cuda")
    h = room[:T * B * H].view(T, B, H)
    d = room.view(T, B, 4 * H)
    state = room[-B * H:].view(B, H)
    in_h = h.view(-1)[5:5 + B * H].view(B, H)
    lengths = room[4:4 + B].view(torch.int32)
    grad = torch.zeros(T, B, H, device="cuda", requires_grad=True)
    # 2^31 channels of one step would do, but not of 17, which are 3 waves of
    # 64 for each 64 channels: no such tensor is made
    wide = torch.empty(1, 1, 4 * 32767, device="cuda").expand(17, 65536, -1)
    for call in (
            lambda: G.glr_forward(gates, in_h, out=h),
            lambda: G.glr_forward(gates, c0, lengths, out=h),
            lambda: G.glr_forward(gates, c0, out=grad),
            lambda: G.glr_backward(dh, state, gates, c0, marks, out=d),
            lambda: G.glr_backward(dh, dcT, gates, c0, marks, lengths, out=d),
            lambda: G.glr_backward(h, dcT, gates, c0, marks, out=d),
            lambda: G.glr_backward(
                dh, dcT, gates, c0, room[:marks.numel()].view(marks.shape),
                out=d),
            lambda: G.glr_forward(wide)):
        with pytest.raises(RuntimeError, match="glr"):
            call()
    assert not room.any()
    want = G.glr_forward(gates, c0)[0]
    assert torch.equal(G.glr_forward(gates, c0, out=h)[0], want)
    with torch.no_grad():
        G.glr_forward(gates, c0, out=grad)
    assert torch.equal(grad.detach(), want)


@GPU
def test_step_in_inference_mode():
    gates, c0, *_ = make(1, 3, 70, torch.float32, "cuda")
    c = c0.clone()
    want = G.glr_step(gates[0], c)
    with torch.inference_mode():
        state = c0.clone()
        assert torch.equal(G.glr_step(gates[0], state), want)
        assert torch.equal(state, c)


@GPU
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,B,H", [(129, 17, 1001), (300, 33, 500),
                                   (450, 16, 1024)])
def test_windows_of_many_channels(T, B, H, dtype):
    """Over 128 steps of over 16384 channels, in shorter tiles: whole rows
    and rows that end anywhere, twice with the same bits."""
    for ragged in (False, True):
        gates, c0, dh, dcT, lengths = make(T, B, H, dtype, "cuda",
                                           ragged=ragged)
        h, cT, dgates, dc0 = check(gates, c0, dh, dcT, lengths)
        again = G.glr_forward(gates, c0, lengths, training=True)
        assert torch.equal(again[0], h) and torch.equal(again[1], cT)
        back = G.glr_backward(dh, dcT, gates, c0, again[2], lengths)
        assert torch.equal(back[0], dgates) and torch.equal(back[1], dc0)


@GPU
def test_tangents_are_refused():
    """The kernels would drop them."""
    import torch.autograd.forward_ad as fwd
    gates, c0, dh, dcT, _ = make(5, 3, 4, torch.float32, "cuda")
    _, _, marks = G.glr_forward(gates, c0, training=True)
    with fwd.dual_level():
        dual = lambda x: fwd.make_dual(x, torch.ones_like(x))  # noqa: E731
        g, c, d, e = (dual(x) for x in (gates, c0, dh, dcT))
        for call in (
                lambda: G.glr(g, c0), lambda: G.glr(gates, c),
                lambda: G.glr(g.clone().requires_grad_(), c0),
                lambda: G.glr_forward(g, c0), lambda: G.glr_forward(gates, c),
                lambda: G.glr_backward(d, dcT, gates, c0, marks),
                lambda: G.glr_backward(dh, e, gates, c0, marks),
                lambda: G.glr_backward(dh, dcT, g, c0, marks),
                lambda: G.glr_step(g[0], c0),
                lambda: G.glr_step(gates[0], c.clone())):
            with pytest.raises(RuntimeError, match="forward|jvp|tangent"):
                call()
        G.glr(gates, c0)  # others beside them are not
