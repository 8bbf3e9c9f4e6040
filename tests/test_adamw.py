"""The AdamW step against its formulas in 64 bits.

Tolerances. m and v are two products and a sum, each rounded, of numbers that
a 32-bit clip factor went into: off by at most 5 half steps of their terms'
magnitudes. The update m / (r root + eps) adds a root, two products, a sum, a
division: with m's and v's errors under 16 half steps of the terms that made
them. p adds two products and a difference. Codes of m are the nearest e4m3
value, off by at most half a code (2^-4 of the value, or 2^-10 below 2^-6);
codes of r are one of the two neighbours, less than a code away (2^-3, 2^-9).
"""

import pytest
import torch

from zaremba_amd.ops import adamw as A
from zaremba_amd.ops import functional as F_ref

GPU = pytest.mark.gpu
HALF = 2.0 ** -24
E4M3 = torch.float8_e4m3fn


def make(sizes, device, bits=32, grad=torch.float32, seed=0, step=7,
         shadows=True):
    gen = torch.Generator().manual_seed(seed)
    r = lambda n, s: torch.randn(n, generator=gen) * s  # noqa: E731
    out = {"params": [r(n, 0.1) for n in sizes],
           "grads": [(r(n, 1.0) * 10.0 ** (k % 5 - 3)).to(grad)
                     for k, n in enumerate(sizes)]}
    ms = [r(n, 0.1) for n in sizes]
    vs = [r(n, 1.0).square() * 1e-2 for n in sizes]
    if bits == 32:
        out["exp_avgs"], out["exp_avg_sqs"] = ms, vs
    else:
        for name, scales, xs in (
                ("exp_avgs", "exp_avg_scales", ms),
                ("exp_avg_sqs", "exp_avg_sq_scales",
                 [v.sqrt() for v in vs])):
            out[name], out[scales] = [], []
            for x in xs:
                b = F_ref._blocks(x)
                s, inv = F_ref._e4m3_scales(b)
                out[scales].append(s)
                out[name].append((b * inv).reshape(-1)[:x.numel()].to(E4M3))
    if shadows:
        out["shadows"] = [p.to(torch.bfloat16) for p in out["params"]]
    out = {k: [x.to(device) for x in v] for k, v in out.items()}
    out["step"] = torch.full((1,), step, dtype=torch.int64, device=device)
    return out


def clone(x):
    return {k: [t.clone() for t in v] if isinstance(v, list) else v.clone()
            for k, v in x.items()}


def value(codes, scales):
    n = codes.numel()
    b = F_ref._blocks(codes.float().double().reshape(-1))
    return (b * scales.double()[:, None]).view(-1)[:n]


def oracle(x, lr, betas, eps, weight_decay, max_norm, grad_scale):
    """(p, m, v), the error scales of m and v, and the norm, in 64 bits."""
    b1, b2 = betas
    t = int(x["step"]) + 1
    gs = [g.double().cpu() for g in x["grads"]]
    norm = torch.sqrt(sum((g ** 2).sum() for g in gs)) * grad_scale
    scale = grad_scale
    if max_norm is not None:
        scale *= min(1.0, max_norm / (float(norm) + 1e-6))
    out = []
    for k, p in enumerate(x["params"]):
        if "exp_avg_scales" in x:
            m = value(x["exp_avgs"][k].cpu(), x["exp_avg_scales"][k].cpu())
            v = value(x["exp_avg_sqs"][k].cpu(),
                      x["exp_avg_sq_scales"][k].cpu()) ** 2
        else:
            m = x["exp_avgs"][k].double().cpu()
            v = x["exp_avg_sqs"][k].double().cpu()
        g = gs[k] * scale
        size_m = b1 * m.abs() + (1 - b1) * g.abs()
        m = b1 * m + (1 - b1) * g
        v = b2 * v + (1 - b2) * g * g
        denom = torch.sqrt(v / (1 - b2 ** t)) + eps
        rate = lr / (1 - b1 ** t)
        p = p.double().cpu() * (1 - lr * weight_decay) - rate * m / denom
        out.append((p, m, v, size_m, rate * size_m / denom))
    return out, norm


def close(got, want, size, halves, name):
    got = got.double().cpu().reshape(-1)
    off = (got - want.reshape(-1)).abs()
    allowed = size.reshape(-1) * halves * HALF + 1e-37
    assert bool((off <= allowed).all()), (name, float((off - allowed).max()))


KW = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1,
          max_norm=0.5, grad_scale=1.0)


def check(x, **kw):
    kw = {**KW, **kw}
    want, norm = oracle(x, **kw)
    t = int(x["step"])
    got = A.adamw_step_(x["params"], x["grads"], x["exp_avgs"],
                        x["exp_avg_sqs"], x["step"],
                        exp_avg_scales=x.get("exp_avg_scales"),
                        exp_avg_sq_scales=x.get("exp_avg_sq_scales"),
                        shadows=x.get("shadows"), **kw)
    assert int(x["step"]) == t + 1
    if kw["max_norm"] is None:
        assert got is None
    else:
        assert got.shape == () and got.dtype == torch.float32
        assert abs(float(got) - float(norm)) <= 2 * HALF * float(norm)
    for k, (p, m, v, size_m, move) in enumerate(want):
        close(x["params"][k], p, p.abs() + KW["lr"] * 0 + move, 24, "p")
        if x.get("shadows") is not None and x["shadows"][k] is not None:
            assert torch.equal(x["shadows"][k],
                               x["params"][k].to(torch.bfloat16))
        if "exp_avg_scales" not in x:
            close(x["exp_avgs"][k], m, size_m, 8, "m")
            close(x["exp_avg_sqs"][k], v, v, 8, "v")
            continue
        for name, w, part in (("exp_avg", m, 1), ("exp_avg_sq", v.sqrt(), 2)):
            codes = x[name + "s"][k].cpu()
            scales = x[name + "_scales"][k].cpu()
            amax = F_ref._blocks(w).abs().amax(1)
            # m's two parts may cancel: its roundings are of their sizes
            size = F_ref._blocks(size_m if part == 1 else w).abs().amax(1)
            close(scales, torch.where(amax < 2.0 ** -100, 0 * amax,
                                      amax / 448), size / 448, 16, name)
            have = value(codes, scales)
            s = scales.double().repeat_interleave(256)[:w.numel()]
            step = torch.maximum(w.abs() * 2.0 ** -4, s * 2.0 ** -10) * part
            slack = (size_m if part == 1 else w) * 16 * HALF
            assert bool(((have - w).abs() <= step + slack + 1e-37).all()), name
            if part == 2:
                # a root that is not zero is not stored as zero
                assert bool(((have > 0) | (w == 0) | (s == 0)).all())
                assert bool((have >= 0).all())
    return x


SIZES = [[1], [3, 256, 257], [1000, 1, 255, 4096], [20000, 17, 70001]]


@pytest.mark.parametrize("bits", [32, 8])
def test_eager_matches_oracle(bits):
    for sizes in SIZES:
        check(make(sizes, "cpu", bits))
        check(make(sizes, "cpu", bits, torch.bfloat16), max_norm=None)
        check(make(sizes, "cpu", bits, step=0), max_norm=1e9, grad_scale=0.25)


def test_draw_is_right_in_the_mean():
    """E[value^2] = x^2 over even draws, and the two neighbours only."""
    x = torch.cat([torch.rand(300) * 448, torch.rand(200) * 2.0 ** -5,
                   torch.tensor([0.0, 448.0, 2.0 ** -6, 2.0 ** -9])])
    n = 4096
    u = (torch.arange(n).float() + 0.5) / n
    codes = F_ref.draw_e4m3(x[:, None].expand(-1, n).contiguous(),
                            u[None].expand(x.numel(), -1).contiguous())
    got = codes.view(E4M3).double()
    spread = got.square().amax(1) - got.square().amin(1)
    off = got.square().mean(1) - x.double() ** 2
    fine = x >= 2.0 ** -9   # below, the mean is held up on purpose
    # n even draws hit a share of them within 1 / n
    assert bool((off.abs() <= spread / n + 1e-6 * x ** 2)[fine].all())
    assert bool((off >= -spread / n - 1e-6 * x ** 2).all())
    assert int((codes.amax(1) - codes.amin(1)).max()) == 1


@pytest.mark.parametrize("bits", [32, 8])
def test_lists_that_do_not_fit_are_refused_unchanged(bits):
    """On the CPU as on the GPU: a gradient of one value is not spread over
    its parameter, and nothing has moved when a list turns out wrong."""
    names = ("params", "grads", "exp_avgs", "exp_avg_sqs")
    scales = ("exp_avg_scales", "exp_avg_sq_scales")

    def refused(change):
        x = make([10, 300], "cpu", bits)
        y = clone(x)
        change(y)
        keep = clone(y)
        with pytest.raises(RuntimeError, match="adamw"):
            A.adamw_step_(*(y[name] for name in names), y["step"], lr=0.1,
                          shadows=y["shadows"],
                          **{name: y.get(name) for name in scales})
        for name, a in y.items():
            b = keep[name]
            for t, u in zip(a, b) if isinstance(a, list) else [(a, b)]:
                assert torch.equal(t.float(), u.float()), name

    def put(name, k, f):
        return lambda x: x[name].__setitem__(k, f(x[name][k]))

    for name in names + ("shadows",) + (scales if bits == 8 else ()):
        refused(put(name, 1, lambda t: t[:1]))
        refused(lambda x: x[name].pop())
    for name in ("params", "exp_avgs", "exp_avg_sqs"):
        refused(put(name, 1, lambda t: t.view(torch.uint8).repeat(2)
                    [::2].view(t.dtype) if t.dtype == E4M3
                    else t.repeat(2)[::2]))
    refused(lambda x: x.update(step=x["step"].float()))
    refused(lambda x: x.update(step=torch.zeros(2, dtype=torch.int64)))
    refused(lambda x: x["params"].__setitem__(0, x["params"][1][:10]))
    if bits == 8:
        for name in scales:
            refused(lambda x: x.pop(name))
    else:
        refused(lambda x: x.update(exp_avg_sq_scales=[torch.zeros(1),
                                                      torch.zeros(2)]))


@pytest.mark.parametrize("eps", [1e-50, 2.0 ** -127, float("nan")])
def test_eps_that_float32_does_not_hold_is_refused(eps):
    x = make([5], "cpu")
    with pytest.raises(ValueError, match="eps"):
        A.adamw_step_(x["params"], x["grads"], x["exp_avgs"],
                      x["exp_avg_sqs"], x["step"], lr=0.1, eps=eps)
    with pytest.raises(ValueError, match="eps"):
        A.AdamW([torch.zeros(3)], eps=eps)


def least_eps(device, bits):
    x = make([300], device, bits, step=0, shadows=False)
    for name in ("grads", "exp_avgs", "exp_avg_sqs"):
        x[name][0].view(torch.uint8).zero_()
    p = x["params"][0].clone()
    for _ in range(2):
        A.adamw_step_(x["params"], x["grads"], x["exp_avgs"],
                      x["exp_avg_sqs"], x["step"], lr=0.1, eps=2.0 ** -126,
                      weight_decay=0.0,
                      exp_avg_scales=x.get("exp_avg_scales"),
                      exp_avg_sq_scales=x.get("exp_avg_sq_scales"))
    assert torch.equal(x["params"][0], p)     # 0 / eps


@pytest.mark.parametrize("bits", [32, 8])
def test_least_eps_divides_zero(bits):
    least_eps("cpu", bits)


@GPU
@pytest.mark.parametrize("bits", [32, 8])
def test_least_eps_divides_zero_gpu(bits):
    least_eps("cuda", bits)


@pytest.mark.parametrize("seed", [0, 2, 10, 45, 62, 165])
def test_draw_is_right_between_its_neighbours(seed):
    """The same at values that lie so near a code that 4096 even draws may
    all give it, and anywhere else: off by one draw of the gap between the
    neighbours, not of the codes that were drawn."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.cat([torch.rand(300, generator=gen) * 448,
                   torch.rand(200, generator=gen) * 2.0 ** -5 + 2.0 ** -9])
    value = torch.arange(127, dtype=torch.uint8).view(E4M3).float()
    near = value[2:126, None] * (1 + torch.tensor([[-1e-5, -1e-6, 0, 1e-6,
                                                    1e-5]]))
    x = torch.cat([x, near.flatten()])
    low = torch.searchsorted(value, x, right=True) - 1
    a, b = value[low].double(), value[(low + 1).clamp(max=126)].double()
    n = 4096
    u = (torch.arange(n).float() + 0.5) / n
    codes = F_ref.draw_e4m3(x[:, None].expand(-1, n).contiguous(),
                            u[None].expand(x.numel(), -1).contiguous())
    assert bool(((codes == low[:, None]) | (codes == low[:, None] + 1)).all())
    off = codes.view(E4M3).double().square().mean(1) - x.double() ** 2
    assert bool((off.abs() <= (b * b - a * a) / n + 1e-6 * x ** 2).all())


def test_hash_is_even():
    u = F_ref.hash_uniform(torch.arange(1 << 16), 12345)
    # 65536 draws: the mean of uniforms is within 5 sigma = 5 * 0.289 / 256
    assert abs(float(u.mean()) - 0.5) < 5 * 0.289 / 256
    assert float(u.min()) >= 0 and float(u.max()) < 1
    other = F_ref.hash_uniform(torch.arange(1 << 16), 12346)
    both = float(((u - 0.5) * (other - 0.5)).mean()) * 12
    assert abs(both) < 5 / 256


def test_eight_bit_average_moves():
    """v in 8 bits follows a gradient that grows tenfold, which the nearest
    code would not at b2 = 0.999."""
    n = 4096
    x = make([n], "cpu", 8, shadows=False)
    x["exp_avg_sqs"][0].copy_(torch.full((n,), 64.0))
    x["exp_avg_sqs"][0][::256] = 448.0
    x["exp_avg_sq_scales"][0].fill_(1.0)
    g = torch.full((n,), 100.0)
    g[::256] = 448.0
    x["grads"] = [g]
    before = 64.0 ** 2
    for _ in range(200):
        A.adamw_step_(x["params"], x["grads"], x["exp_avgs"],
                      x["exp_avg_sqs"], x["step"], lr=0.0,
                      betas=(0.9, 0.999),
                      exp_avg_scales=x["exp_avg_scales"],
                      exp_avg_sq_scales=x["exp_avg_sq_scales"])
    keep = torch.ones(n, dtype=torch.bool)
    keep[::256] = False
    v = value(x["exp_avg_sqs"][0], x["exp_avg_sq_scales"][0])[keep].square()
    want = before * 0.999 ** 200 + 1e4 * (1 - 0.999 ** 200)
    # each of 200 draws moves v by at most one code (25 %) with a chance of
    # its drift (under 0.6 % of v) over that: the sum's deviation is under
    # sqrt(200 * 0.006 * 0.25) = 55 % of v for one element, 0.9 % for the
    # mean of 4080; 5 of those
    assert abs(float(v.mean()) / want - 1) < 0.045


def refusals(device):
    def call(change, **kw):
        x = make([10, 300], device)
        change(x)
        x = {**x, **kw}
        return lambda: A.adamw_step_(
            x["params"], x["grads"], x["exp_avgs"], x["exp_avg_sqs"],
            x["step"], lr=x.get("lr", 0.1), betas=x.get("betas", (0.9, 0.99)),
            eps=x.get("eps", 1e-8), weight_decay=x.get("wd", 0.0),
            max_norm=x.get("max_norm"), shadows=x["shadows"],
            grad_scale=x.get("grad_scale", 1.0),
            exp_avg_scales=x.get("exp_avg_scales"))

    nothing = lambda x: None  # noqa: E731
    return [call(nothing, lr=-1.0), call(nothing, betas=(0.9, 1.0)),
            call(nothing, eps=0.0), call(nothing, wd=-1.0),
            call(nothing, max_norm=0.0), call(nothing, lr=float("nan")),
            call(nothing, grad_scale=0.0), call(nothing, grad_scale=-1.0),
            call(nothing, exp_avg_scales=[torch.zeros(1, device=device)] * 2),
            call(nothing, params=[]), call(lambda x: x["grads"].pop()),
            call(lambda x: x["shadows"].pop())]


def test_refusals_eager():
    for call in refusals("cpu"):
        with pytest.raises((ValueError, RuntimeError), match="adamw"):
            call()
    with pytest.raises(ValueError):
        A.AdamW([torch.zeros(3)], bits=16)
    with pytest.raises(ValueError):
        A.AdamW([])


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_round_trip(bits):
    torch.manual_seed(0)
    p = [torch.nn.Parameter(torch.randn(300)), torch.nn.Parameter(
        torch.randn(3, 5))]
    q = [torch.nn.Parameter(x.detach().clone()) for x in p]
    a, b = A.AdamW(p, bits=bits), A.AdamW(q, bits=bits)

    def step(opt, params, seed):
        gen = torch.Generator().manual_seed(seed)
        for x in params:
            x.grad = torch.randn(x.shape, generator=gen)
        opt.step(0.01, 1.0)

    step(a, p, 1)
    step(b, q, 1)
    c = A.AdamW(q, bits=bits)
    c.load_state_dict(b.state_dict())
    step(a, p, 2)
    step(c, q, 2)
    assert all(torch.equal(x, y) for x, y in zip(p, q))
    with pytest.raises(ValueError):
        A.AdamW(p, bits=40 - bits).load_state_dict(a.state_dict())
    with pytest.raises(ValueError):
        A.AdamW(p[:1], bits=bits).load_state_dict(a.state_dict())
    # a parameter without a gradient stays as it is
    keep = p[1].detach().clone()
    p[1].grad = None
    a.step(0.01)
    assert torch.equal(p[1], keep)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_saved_state_stays_as_it_was(bits):
    """Going back to it after more steps gives the same steps again."""
    torch.manual_seed(0)
    p = torch.nn.Parameter(torch.randn(300))
    opt = A.AdamW([p], bits=bits)

    def steps():
        gen = torch.Generator().manual_seed(3)
        for _ in range(3):
            p.grad = torch.randn(300, generator=gen)
            opt.step(0.01, 1.0)
        return p.detach().clone()

    steps()
    saved, start = opt.state_dict(), p.detach().clone()
    first = steps()
    opt.load_state_dict(saved)
    p.data.copy_(start)
    assert torch.equal(steps(), first)


@pytest.mark.parametrize("bits,name", [
    (32, "exp_avg_sqs"), (8, "exp_avg_sqs"), (8, "exp_avg_sq_scales")])
def test_states_of_another_model_change_nothing(bits, name):
    p = torch.nn.Parameter(torch.randn(300))
    opt = A.AdamW([p], bits=bits)
    p.grad = torch.randn(300)
    opt.step(0.01)
    other, keep = opt.state_dict(), opt.state_dict()
    p.grad = torch.randn(300)
    for x in other["exp_avgs"]:
        x.view(torch.uint8).fill_(1)
    other[name] = [x[:1] for x in other[name]]
    with pytest.raises(ValueError, match=name):
        opt.load_state_dict(other)
    for a, b in zip(opt.state_dict()["exp_avgs"], keep["exp_avgs"]):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


# ---------------------------------------------------------------------------
# kernels
# ---------------------------------------------------------------------------

@GPU
def test_refusals_gpu():
    for call in refusals("cuda"):
        with pytest.raises((ValueError, RuntimeError), match="adamw"):
            call()

    def refused(change):
        x = make([10, 300], "cuda")
        change(x)
        with pytest.raises(RuntimeError, match="adamw"):
            A.adamw_step_(x["params"], x["grads"], x["exp_avgs"],
                          x["exp_avg_sqs"], x["step"], lr=0.1,
                          shadows=x["shadows"])

    def put(name, k, f):
        def change(x):
            x[name][k] = f(x[name][k])
        return change

    for name in ("params", "grads", "exp_avgs", "exp_avg_sqs", "shadows"):
        refused(put(name, 1, lambda t: t[:299]))
        refused(put(name, 1, lambda t: t.cpu()))
        refused(put(name, 1, lambda t: t.half()))
        refused(put(name, 1, lambda t: t.repeat(2)[::2]))
    refused(lambda x: x.update(step=x["step"].int()))
    refused(lambda x: x.update(step=x["step"].cpu()))
    # the same tensor twice, and two that overlap
    refused(lambda x: x["params"].__setitem__(0, x["params"][1][:10]))
    refused(lambda x: x["exp_avgs"].__setitem__(0, x["exp_avg_sqs"][1][5:15]))
    x = make([300], "cuda", 8)
    x["exp_avg_scales"][0] = x["exp_avg_scales"][0][:1]
    with pytest.raises(RuntimeError, match="adamw"):
        A.adamw_step_(x["params"], x["grads"], x["exp_avgs"],
                      x["exp_avg_sqs"], x["step"], lr=0.1,
                      exp_avg_scales=x["exp_avg_scales"],
                      exp_avg_sq_scales=x["exp_avg_sq_scales"])


@GPU
@pytest.mark.parametrize("grad", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
def test_kernels_match_oracle(bits, grad):
    for sizes in SIZES:
        check(make(sizes, "cuda", bits, grad))
        check(make(sizes, "cuda", bits, grad, shadows=False), max_norm=None)
        check(make(sizes, "cuda", bits, grad, step=0), max_norm=1e9,
              grad_scale=0.25)
        check(make(sizes, "cuda", bits, grad, step=100000), max_norm=1e-3,
              betas=(0.0, 0.999), weight_decay=0.0)


@GPU
@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_and_empty_ones(bits):
    """More tensors than a launch takes, and some that hold nothing."""
    sizes = [(k * 7919) % 1500 for k in range(131)]
    assert 0 in sizes
    x = check(make(sizes, "cuda", bits))
    check(x, grad_scale=3.0)
    x = make([0, 0], "cuda", bits)
    check(x)


@GPU
@pytest.mark.parametrize("bits", [32, 8])
def test_no_alignment_and_some_shadows(bits):
    """Tensors that begin anywhere, with guards around them."""
    for shift in (1, 2, 3):
        x = make([1027, 5, 600], "cuda", bits)
        rooms = []
        for name, list_ in x.items():
            if name == "step":
                continue
            for k, t in enumerate(list_):
                byte = t.dtype == E4M3
                room = torch.full((t.numel() + 16,), 3, device="cuda",
                                  dtype=torch.uint8 if byte else t.dtype)
                at = room[shift:shift + t.numel()]
                at.copy_(t.view(torch.uint8) if byte else t)
                list_[k] = at.view(E4M3) if byte else at
                rooms.append((room, t.numel()))
        x["shadows"][1] = None
        check(x)
        for room, n in rooms:
            assert bool((room[:shift] == 3).all())
            assert bool((room[shift + n:] == 3).all())


@GPU
@pytest.mark.parametrize("grad", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
def test_kernels_follow_eager(bits, grad):
    """Ten steps on both sides. In 8 bits a code next to a border may differ
    where the clip factor does in its last bit: none of them more than one
    code, and fewer than one in 10^4."""
    x = make([5000, 70000, 33], "cuda", bits, grad)
    y = {k: [t.cpu() for t in v] if isinstance(v, list) else v.cpu()
         for k, v in clone(x).items()}
    gen = torch.Generator().manual_seed(5)
    for _ in range(10):
        for side in (x, y):
            A.adamw_step_(side["params"], side["grads"], side["exp_avgs"],
                          side["exp_avg_sqs"], side["step"],
                          exp_avg_scales=side.get("exp_avg_scales"),
                          exp_avg_sq_scales=side.get("exp_avg_sq_scales"),
                          shadows=side["shadows"], **KW)
        if bits == 8:
            for name in ("exp_avgs", "exp_avg_sqs"):
                for a, b in zip(x[name], y[name]):
                    a, b = a.cpu().view(torch.uint8), b.view(torch.uint8)
                    d = (a.int() - b.int()).abs()
                    assert float((d > 0).float().mean()) <= 1e-4
                    b.copy_(a)  # go on from the same codes
                for a, b in zip(x[name[:-1] + "_scales"],
                                y[name[:-1] + "_scales"]):
                    b.copy_(a)
        for a, b in zip(x["params"], y["params"]):
            # ten steps of at most lr times a few, each 24 half steps off
            assert float((a.cpu() - b).abs().max()) < 10 * 24 * HALF
        for k, g in enumerate(x["grads"]):
            new = (torch.randn(g.shape, generator=gen) * 0.1).to(g.dtype)
            g.copy_(new)
            y["grads"][k].copy_(new)


@GPU
@pytest.mark.parametrize("bits", [32, 8])
def test_zeros_and_extremes(bits):
    n = 600
    x = make([n], "cuda", bits, step=0, shadows=False)
    for name in ("exp_avgs", "exp_avg_sqs"):
        x[name][0].view(torch.uint8).zero_()
    x["grads"][0].zero_()
    p = x["params"][0].clone()
    check(x, max_norm=None, weight_decay=0.0)
    assert torch.equal(x["params"][0], p)     # nothing moves on zeros
    for name in ("exp_avgs", "exp_avg_sqs"):
        assert not x[name][0].view(torch.uint8).any()
    # one block of gradients over 10^12 to 10^-9, and one of the tiniest
    g = x["grads"][0]
    g[:256] = torch.logspace(12, -9, 256, device="cuda")
    g[256:512] = 1e-42
    g[512:] = 0
    check(x, max_norm=None, weight_decay=0.0)
    assert bool(torch.isfinite(x["params"][0]).all())
    # the moves are at most the rate's: sqrt(v) was never rounded to zero
    x["grads"][0].zero_()
    before = x["params"][0].clone()
    check(x, max_norm=None, weight_decay=0.0)
    assert float((x["params"][0] - before).abs().max()) < 1.0


@GPU
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_not_finite_is_seen(bad):
    for bits in (32, 8):
        x = make([700], "cuda", bits)
        x["grads"][0][300] = bad
        norm = A.adamw_step_(
            x["params"], x["grads"], x["exp_avgs"], x["exp_avg_sqs"],
            x["step"], lr=0.1, max_norm=1.0,
            exp_avg_scales=x.get("exp_avg_scales"),
            exp_avg_sq_scales=x.get("exp_avg_sq_scales"))
        assert not bool(torch.isfinite(norm))
        assert bool(torch.isnan(x["params"][0][300]))
        if bits == 8:  # and stays seen in the states
            m = value(x["exp_avgs"][0].cpu(), x["exp_avg_scales"][0].cpu())
            assert not bool(torch.isfinite(m[300]))


@GPU
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_and_replayed(bits):
    """Two graphs on states of their own, replayed in turn with eager work
    between: the step count goes on, and the bits are the eager ones."""
    def step(x):
        return A.adamw_step_(
            x["params"], x["grads"], x["exp_avgs"], x["exp_avg_sqs"],
            x["step"], exp_avg_scales=x.get("exp_avg_scales"),
            exp_avg_sq_scales=x.get("exp_avg_sq_scales"),
            shadows=x["shadows"], **KW)

    sides = []
    for seed in (0, 1):
        x = make([3000, 77, 513], "cuda", bits, seed=seed)
        eager = clone(x)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(x)
        torch.cuda.current_stream().wait_stream(side)
        step(eager)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norm = step(x)
        sides.append((x, eager, graph, norm))
    for turn in range(4):
        for x, eager, graph, norm in sides:
            for g, e in zip(x["grads"], eager["grads"]):
                g.mul_(0.7)
                e.mul_(0.7)
            graph.replay()
            want = step(eager)
            torch.cuda.synchronize()
            assert torch.equal(norm, want)
            for name in x:
                a, b = x[name], eager[name]
                for t, u in zip(a, b) if isinstance(a, list) else [(a, b)]:
                    assert torch.equal(t.view(torch.uint8) if
                                       t.dtype == E4M3 else t,
                                       u.view(torch.uint8) if
                                       u.dtype == E4M3 else u), (name, turn)


@GPU
def test_another_stream():
    x = make([100000, 3], "cuda")
    y = clone(x)
    check(x)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        check(y)
    st.synchronize()
    assert torch.equal(x["params"][0], y["params"][0])


@GPU
def test_writes_are_seen_by_autograd():
    x = make([30], "cuda")
    p = x["params"][0].requires_grad_()
    y = (p * p).sum()
    A.adamw_step_(x["params"], x["grads"], x["exp_avgs"], x["exp_avg_sqs"],
                  x["step"], lr=0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()


@GPU
@pytest.mark.parametrize("bits", [32, 8])
def test_a_tensor_of_over_two_to_the_31(bits):
    """Offsets past 32 bits: the last values of a tensor of 2^31 + 300 follow
    those of a short one that holds the same."""
    n, k = (1 << 31) + 300, 300 + 256
    gen = torch.Generator().manual_seed(1)
    tail = {name: torch.randn(k, generator=gen).cuda()
            for name in ("p", "g", "m")}
    big = {name: torch.zeros(n, device="cuda") for name in ("p", "g")}
    for name in ("p", "g"):
        big[name][-k:] = tail[name]
    kind = torch.float32 if bits == 32 else E4M3
    state = lambda n: torch.zeros(  # noqa: E731
        n, dtype=torch.float32 if bits == 32 else torch.uint8,
        device="cuda").view(kind)
    scales = lambda n: None if bits == 32 else [  # noqa: E731
        torch.zeros(-(-n // 256), device="cuda")]

    def run(p, g, n):
        m, v, ms, vs = state(n), state(n), scales(n), scales(n)
        st = torch.zeros(1, dtype=torch.int64, device="cuda")
        norm = A.adamw_step_([p], [g], [m], [v], st, lr=0.1, max_norm=1.0,
                             exp_avg_scales=ms, exp_avg_sq_scales=vs)
        return p[-k:], m[-k:].float(), norm

    a = run(big["p"], big["g"], n)
    # the short tensor ends as the long one does: 300 into a block of 256
    pad = torch.zeros(44 + 212, device="cuda")
    b = run(torch.cat([pad, tail["p"]]), torch.cat([pad, tail["g"]]), 256 + k)
    for u, v in zip(a, b):
        assert torch.equal(u, v)
    assert not bool(big["p"][:-k].any())


@GPU
def test_gradient_in_what_is_written():
    x = make([10, 300], "cuda")
    before = [p.clone() for p in x["params"]]
    for grads in ([x["grads"][0], x["params"][1]],
                  [x["exp_avgs"][1][:10], x["grads"][1]]):
        with pytest.raises(RuntimeError, match="adamw"):
            A.adamw_step_(x["params"], grads, x["exp_avgs"], x["exp_avg_sqs"],
                          x["step"], lr=0.1)
    assert all(torch.equal(a, b) for a, b in zip(x["params"], before))
    # two parameters may have one gradient
    one = torch.cat([x["grads"][1], x["grads"][0]])
    A.adamw_step_(x["params"], [one[:10], one[:300]], x["exp_avgs"],
                  x["exp_avg_sqs"], x["step"], lr=0.1)
    assert not any(torch.equal(a, b) for a, b in zip(x["params"], before))


@GPU
def test_zeros_among_others_stay_zeros():
    """Rows that no token reads have no gradient: beside others, alone in a
    block of 256, and throughout. Without a clip both sides agree in bits."""
    gen = torch.Generator().manual_seed(3)
    x = make([3000, 512], "cpu", 8, shadows=False)
    for k, n in enumerate((3000, 512)):
        for name in ("exp_avgs", "exp_avg_sqs"):
            x[name][k].view(torch.uint8).zero_()
        keep = torch.rand(n, generator=gen) < 0.5
        keep[256:512] = False
        keep[300 + 4 * k] = True
        x["grads"][k] = torch.where(keep, x["grads"][k], torch.zeros(n))
    y = {k: [t.cuda() for t in v] if isinstance(v, list) else v.cuda()
         for k, v in clone(x).items()}
    for side in (x, y):
        A.adamw_step_(side["params"], side["grads"], side["exp_avgs"],
                      side["exp_avg_sqs"], side["step"], lr=1e-2,
                      exp_avg_scales=side["exp_avg_scales"],
                      exp_avg_sq_scales=side["exp_avg_sq_scales"])
    for k, g in enumerate(x["grads"]):
        for name in ("exp_avgs", "exp_avg_sqs"):
            codes = y[name][k].cpu().view(torch.uint8)
            assert torch.equal(codes, x[name][k].view(torch.uint8)), name
            assert not codes[g == 0].any()
        assert bool((y["exp_avg_sqs"][k].cpu().float()[g != 0] > 0).all())
