"""The gated linear recurrence and AdamW together, as a model's training and
evaluation use them."""

import json
import os
import subprocess
import sys

import pytest
import torch

from zaremba_amd import trainer
from zaremba_amd.checkpoint import (build_model_from_checkpoint,
                                    save_checkpoint)
from zaremba_amd.models.lstm_lm import Model
from zaremba_amd.ops.adamw import AdamW
from zaremba_amd.ops import functional as F_ref

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
GPU = pytest.mark.gpu


def model(engine="eager", vocab=60, hidden=24, layers=2, dropout=0.0,
          seed=0, **kw):
    torch.manual_seed(seed)
    return Model(vocab, hidden, layers, dropout, 0.1, engine=engine,
                 cell="glr", **kw)


def batch(T, B, vocab, seed=1, device="cpu"):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randint(0, vocab, (T, B), generator=gen).to(device),
            torch.randint(0, vocab, (T, B), generator=gen).to(device))


def test_unknown_cell_is_refused():
    with pytest.raises(ValueError, match="cell"):
        Model(10, 4, 1, 0.0, 0.1, cell="gru")


def test_model_is_its_formulas():
    """Scores of the model against the cell written out step by step."""
    m = model().double()
    x, y = batch(7, 3, 60)
    states = [(h.double(), c.double()) for h, c in m.state_init(3)]
    scores, states = m(x, states)
    cur = m.embed.W[x]
    for k, layer in enumerate(m.rnns):
        c, out = torch.zeros(3, 24, dtype=torch.float64), []
        for t in range(7):
            g = cur[t] @ layer.W_x.t() + layer.b_x
            i, f, o, n = (g[:, j * 24:(j + 1) * 24] for j in range(4))
            c = torch.sigmoid(f) * c + torch.sigmoid(i) * torch.tanh(n)
            out.append(torch.sigmoid(o) * torch.tanh(c))
        cur = torch.stack(out)
        # a dozen roundings of 2^-53 of numbers under 1
        assert float((states[k][1] - c).detach().abs().max()) < 1e-14
    want = cur.view(21, -1) @ m.fc.W.t() + m.fc.b
    assert float((scores - want).detach().abs().max()) < 1e-13


def test_windows_carry_the_state():
    m = model().eval()
    x, _ = batch(12, 3, 60)
    with torch.no_grad():
        whole, _ = m(x, m.state_init(3))
        states, parts = m.state_init(3), []
        for a, b in ((0, 5), (5, 6), (6, 12)):
            s, states = m(x[a:b], states)
            parts.append(s)
    # the projection's sums may run in another order: 24 terms under 1
    assert float((torch.cat(parts) - whole).abs().max()) < 24 * 2.0 ** -23


@pytest.mark.parametrize("bits", [32, 8])
def test_checkpoint_carries_cell_and_states(tmp_path, bits):
    m = model()
    opt = AdamW(m.parameters(), bits=bits)

    def steps(mm, oo, seeds):
        mm.train()
        for s in seeds:
            x, y = batch(6, 3, 60, seed=s)
            mm.zero_grad()
            scores, _ = mm(x, mm.state_init(3))
            trainer.nll_loss(scores, y).backward()
            trainer.adamw_step(mm, oo, 1e-2, 5.0)

    steps(m, opt, (1, 2))
    path = str(tmp_path / "m.pt")
    save_checkpoint(path, m, extra={"optimizer": opt.state_dict()})
    m2, payload = build_model_from_checkpoint(path, engine="eager")
    assert m2.cell == "glr"
    opt2 = AdamW(m2.parameters(), bits=bits)
    opt2.load_state_dict(payload["optimizer"])
    steps(m, opt, (3, 4))
    steps(m2, opt2, (3, 4))
    for a, b in zip(m.parameters(), m2.parameters()):
        assert torch.equal(a, b)


def test_checkpoint_without_cell_is_an_lstm(tmp_path):
    m = Model(20, 8, 1, 0.0, 0.1, engine="eager")
    path = str(tmp_path / "m.pt")
    save_checkpoint(path, m)
    payload = torch.load(path, weights_only=False)
    del payload["model_args"]["cell"]
    torch.save(payload, path)
    m2, _ = build_model_from_checkpoint(path, engine="eager")
    assert m2.cell == "lstm"


def run_cli(args):
    return subprocess.run([sys.executable] + args, cwd=REPO, timeout=300,
                          capture_output=True, text=True)


@pytest.mark.timeout(300)
@pytest.mark.parametrize("optimizer", ["adamw", "adamw8bit"])
def test_cli_trains_saves_and_resumes(tmp_path, optimizer):
    ck, jl = str(tmp_path / "m.pt"), str(tmp_path / "m.jsonl")
    args = ["main.py", "--device", "cpu", "--data",
            "synthetic:vocab=40,tokens=3000", "--hidden_size", "16",
            "--layer_num", "2", "--seq_length", "8", "--batch_size", "4",
            "--dropout", "0.1", "--seed", "1", "--cell", "glr",
            "--optimizer", optimizer, "--learning_rate", "0.005"]
    r = run_cli(args + ["--total_epochs", "1", "--save", ck, "--jsonl", jl])
    assert r.returncode == 0, r.stderr[-2000:]
    assert "Test set perplexity" in r.stdout
    assert any(json.loads(line)["event"] == "final" for line in open(jl))
    r = run_cli(args + ["--total_epochs", "2", "--resume", ck])
    assert r.returncode == 0, r.stderr[-2000:]
    assert "Resumed from" in r.stdout
    # states of the other kind are refused
    other = "adamw" if optimizer == "adamw8bit" else "adamw8bit"
    args[args.index(optimizer)] = other
    r = run_cli(args + ["--total_epochs", "2", "--resume", ck])
    assert r.returncode != 0 and "bits" in r.stderr


@pytest.mark.timeout(300)
def test_cli_refuses_states_that_were_not_saved(tmp_path):
    ck = str(tmp_path / "m.pt")
    args = ["main.py", "--device", "cpu", "--data",
            "synthetic:vocab=40,tokens=3000", "--hidden_size", "16",
            "--layer_num", "1", "--seq_length", "8", "--batch_size", "4"]
    r = run_cli(args + ["--total_epochs", "1", "--save", ck])
    assert r.returncode == 0, r.stderr[-2000:]
    r = run_cli(args + ["--total_epochs", "2", "--resume", ck,
                        "--optimizer", "adamw"])
    assert r.returncode != 0 and "no optimizer states" in r.stderr


@pytest.mark.timeout(300)
def test_cli_does_not_drop_states(tmp_path):
    """An AdamW run that is resumed without naming AdamW."""
    ck = str(tmp_path / "m.pt")
    args = ["main.py", "--device", "cpu", "--data",
            "synthetic:vocab=40,tokens=1500", "--hidden_size", "8",
            "--layer_num", "1", "--seq_length", "8", "--batch_size", "4"]
    r = run_cli(args + ["--total_epochs", "1", "--optimizer", "adamw",
                        "--save", ck])
    assert r.returncode == 0, r.stderr[-2000:]
    r = run_cli(args + ["--total_epochs", "2", "--resume", ck])
    assert r.returncode != 0 and "saved under AdamW" in r.stderr


@pytest.mark.timeout(300)
def test_ensemble_cli(tmp_path):
    r = run_cli(["ensemble.py", "--device", "cpu", "--data",
                 "synthetic:vocab=40,tokens=3000", "--hidden_size", "16",
                 "--layer_num", "1", "--seq_length", "8", "--batch_size",
                 "4", "--total_epochs", "1", "--ensemble_num", "2", "--cell",
                 "glr", "--optimizer", "adamw", "--learning_rate", "0.01",
                 "--save_dir", str(tmp_path)])
    assert r.returncode == 0, r.stderr[-2000:]
    assert "Test set perplexity of 2 averaged models" in r.stdout


# ---------------------------------------------------------------------------
# HIP engine
# ---------------------------------------------------------------------------

def rel(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return float((a - b).norm() / b.norm())


# bf16 on the way: embedding, gates and h of two layers, weights, scores'
# operands. Each rounding is off by 2^-9 / sqrt(3) of its value in the mean,
# a dozen of them add up to 0.4 %, and the gates' slopes at most double that;
# a gradient passes as many roundings again.
SCORES, GRADS = 1e-2, 2e-2


def _grads_of(m, seed, states):
    x, y = batch(5, 3, 60, seed=seed)
    scores, states = m(x, [(h.detach(), c.detach()) for h, c in states])
    F_ref.nll_loss(scores, y).backward()
    return states


def _rank_main(rank, world, init_file, bits, q):
    import torch.distributed as td
    from zaremba_amd.parallel.bucketer import GradBucketer
    torch.set_num_threads(1)
    td.init_process_group("gloo", init_method=f"file://{init_file}",
                          rank=rank, world_size=world)
    m = model()
    dp = GradBucketer(m, bucket_bytes=4096)
    opt, states = AdamW(m.parameters(), bits=bits), m.state_init(3)
    for step in range(3):
        dp.zero_grad()
        states = _grads_of(m, 10 * step + rank, states)
        dp.finalize_backward()
        trainer.adamw_step(m, opt, 1e-2, 0.5)
    q.put((rank, [p.detach().numpy().copy() for p in m.parameters()]))
    td.destroy_process_group()


@pytest.mark.timeout(180)
@pytest.mark.parametrize("bits", [32, 8])
def test_ranks_step_alike(tmp_path, bits):
    """Two ranks with a batch each stay one model: the one that takes both
    batches. A sum of two gradients has one rounding in either order."""
    import torch.multiprocessing as mp
    ctx = mp.get_context("spawn")
    q = ctx.SimpleQueue()
    procs = [ctx.Process(target=_rank_main, args=(
        r, 2, str(tmp_path / "pg"), bits, q)) for r in range(2)]
    for p in procs:
        p.start()
    got = dict(q.get() for _ in procs)
    for p in procs:
        p.join(60)
        assert p.exitcode == 0
    threads = torch.get_num_threads()
    torch.set_num_threads(1)
    try:
        m = model()
        opt = AdamW(m.parameters(), bits=bits)
        states = [m.state_init(3) for _ in range(2)]
        for step in range(3):
            m.zero_grad()
            states = [_grads_of(m, 10 * step + r, states[r])
                      for r in range(2)]
            trainer.adamw_step(m, opt, 1e-2, 0.5)
    finally:
        torch.set_num_threads(threads)
    for a, b, p in zip(got[0], got[1], m.parameters()):
        assert torch.equal(torch.from_numpy(a), torch.from_numpy(b))
        assert torch.equal(torch.from_numpy(a), p.detach())


@GPU
@pytest.mark.parametrize("T,B,H", [(35, 20, 200), (9, 40, 64), (700, 2, 72)])
def test_hip_model_follows_eager(T, B, H):
    eager = model(vocab=500, hidden=H).cuda()
    hip = model("hip", vocab=500, hidden=H).cuda()
    hip.load_state_dict(eager.state_dict())
    x, y = batch(T, B, 500, device="cuda")
    out = []
    for m in (eager, hip):
        m.train()
        states = m.state_init(B)
        gen = torch.Generator().manual_seed(3)
        for k, (h, c) in enumerate(states):
            c.copy_(torch.randn(c.shape, generator=gen))
        scores, states = m(x, states)
        loss = F_ref.nll_loss(scores, y)
        loss.backward()
        out.append((scores, states, [p.grad for p in m.parameters()]))
    (s0, st0, g0), (s1, st1, g1) = out
    assert rel(s1, s0) < SCORES
    for (_, c0), (_, c1) in zip(st0, st1):
        assert rel(c1, c0) < SCORES
    for (name, _), a, b in zip(eager.named_parameters(), g1, g0):
        assert rel(a, b) < GRADS, name


@GPU
def test_hip_tokens_one_by_one():
    m = model("hip", vocab=300, hidden=136).cuda().eval()
    x, _ = batch(10, 5, 300, device="cuda")
    with torch.no_grad():
        whole, last = m(x, m.state_init(5))
        want = [c.clone() for _, c in last]
        whole = whole.clone().view(10, 5, -1)
        states = m.state_init(5)
        first = states[0][1]
        for t in range(10):
            s, states = m(x[t:t + 1], states)
            # the same gates, each rounded to bf16; a state's bits may differ
            # where the scan composes its steps in another order, and an h
            # at a border of bf16 with it
            assert rel(s, whole[t]) < 2.0 ** -9
        assert not first.any()          # the caller's state is left alone
    for (_, c), w in zip(states, want):
        assert rel(c, w) < 2.0 ** -9


@GPU
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("cell", ["glr", "lstm"])
def test_hip_adamw_trains(cell, bits):
    """The HIP step against the eager one on the same gradients, and the
    shadows that the next forward reads."""
    torch.manual_seed(0)
    m = Model(203, 72, 2, 0.0, 0.1, engine="hip", cell=cell).cuda()
    opt = AdamW(m.parameters(), bits=bits)
    twin = [p.detach().cpu().clone().requires_grad_() for p in m.parameters()]
    other = AdamW(twin, bits=bits)
    m.train()
    states = m.state_init(4)
    for step in range(3):
        x, y = batch(11, 4, 203, seed=step, device="cuda")
        m.zero_grad(set_to_none=True)
        states = m.detach(states)
        scores, states = m(x, states)
        trainer.nll_loss(scores, y).backward()
        for p, q in zip(m.parameters(), twin):
            q.grad = p.grad.cpu()
        norm = trainer.adamw_step(m, opt, 1e-2, 0.5)
        want = other.step(1e-2, 0.5)
        assert abs(float(norm) - float(want)) <= 2.0 ** -22 * float(want)
        for p, q in zip(m.parameters(), twin):
            # lr times 30 half steps a step (tests/test_adamw.py); in 8 bits
            # a draw next to its border may move a code, 1 / 8 of a value
            off = (p.detach().cpu() - q.detach()).abs()
            if bits == 32:
                assert float(off.max()) < (step + 1) * 32 * 2.0 ** -24
            else:
                assert float((off > 1e-5).float().mean()) < 1e-4
            with torch.no_grad():
                q.copy_(p.cpu())
    m._hip_model.check_aborts()
    before = scores.detach().clone()
    m._hip_model.invalidate_shadows()   # read the masters again
    with torch.no_grad():
        a, _ = m(x, m.state_init(4))
        a = a.clone()
        m._hip_model.refresh_shadows()
        b, _ = m(x, m.state_init(4))
    assert torch.equal(a, b) and not torch.equal(a, before)


@GPU
def test_hip_shadows_are_rewritten():
    m = model("hip", vocab=101, hidden=40).cuda()
    opt = AdamW(m.parameters())
    x, y = batch(5, 3, 101, device="cuda")
    scores, _ = m(x, m.state_init(3))
    trainer.nll_loss(scores, y).backward()
    trainer.adamw_step(m, opt, 1e-1, 1.0)
    hm = m._hip_model
    assert torch.equal(hm.emb_W, m.embed.W.detach().bfloat16())
    assert torch.equal(hm.fc.W, m.fc.W.detach().bfloat16())
    assert torch.equal(hm.fc.WT[:, :101], hm.fc.W.t())
    for rt, layer in zip(hm.layers, m.rnns):
        assert torch.equal(rt.Wx, layer.W_x.detach().bfloat16())
        assert torch.equal(rt.WxT[:, :160], rt.Wx.t())


@GPU
@pytest.mark.parametrize("bits", [32, 8])
def test_training_loop_runs(tmp_path, bits, capsys):
    """trainer.train on the HIP engine, windows, epochs and a checkpoint."""
    from zaremba_amd import data as zdata
    trn, vld, tst, vocab = zdata.synthetic_init(
        vocab_size=50, train_tokens=3000, valid_tokens=600, test_tokens=600,
        seed=1)
    sets = tuple(zdata.minibatch(d, 4, 10) for d in (trn, vld, tst))
    m = model("hip", vocab=vocab, hidden=48, dropout=0.1).cuda()
    opt = AdamW(m.parameters(), bits=bits)
    path = str(tmp_path / "m.pt")
    ppl = trainer.train(sets, m, 2, 1, 5e-3, 1.0, 5.0, 4, save_path=path,
                        optimizer=opt)
    assert ppl == ppl and ppl < 1e4
    assert "Training is over." in capsys.readouterr().out
    m2, payload = build_model_from_checkpoint(path, engine="hip")
    m2.cuda()
    opt2 = AdamW(m2.parameters(), bits=bits)
    opt2.load_state_dict(payload["optimizer"])
    assert int(opt2.step_count) == 2 * len(sets[0])
    for a, b in zip(opt.exp_avgs, opt2.exp_avgs):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@GPU
@pytest.mark.parametrize("T", [1, 9, 200])
@pytest.mark.parametrize("grad", [False, True])
def test_hip_states_stay_as_returned(T, grad):
    """The states of a window are not those of the window after it."""
    m = model("hip", vocab=60, hidden=40).cuda()
    with torch.set_grad_enabled(grad):
        first, kept = None, None
        for seed in (1, 2):
            x, _ = batch(T, 3, 60, seed=seed, device="cuda")
            _, states = m(x, m.state_init(3))
            if first is None:
                first = [(h, c) for h, c in states]
                kept = [(h.clone(), c.clone()) for h, c in states]
    for (h, c), (h0, c0), (h1, c1) in zip(first, kept, states):
        assert torch.equal(h, h0) and torch.equal(c, c0)
        assert not torch.equal(h, h1) and not torch.equal(c, c1)
        assert not h.requires_grad and not c.requires_grad


@GPU
@pytest.mark.parametrize("layers", [1, 2])
@pytest.mark.parametrize("dropout", [0.0, 0.5])
@pytest.mark.parametrize("between", [(9, 4, True), (9, 4, False),
                                     (4, 9, True), (3, 4, False)])
def test_hip_backward_of_an_older_window_is_refused(layers, dropout, between):
    """Its workspaces hold what came between; the newest window's gradients
    are those that it has by itself."""
    T, B, train = between
    m = model("hip", vocab=60, hidden=40, layers=layers,
              dropout=dropout).cuda()

    def window(seed, T, B):
        x, y = batch(T, B, 60, seed=seed, device="cuda")
        scores, _ = m(x, m.state_init(B))
        return trainer.nll_loss(scores, y)

    old = window(1, 9, 4)
    m.train(train)
    with torch.set_grad_enabled(train):
        new = window(2, T, B)
    with pytest.raises(RuntimeError, match="another forward pass"):
        old.backward()
    if not train:
        return
    m.zero_grad()
    new.backward()
    got = [p.grad.clone() for p in m.parameters()]
    if dropout:  # other masks
        return
    m.zero_grad()
    window(2, T, B).backward()
    # the embedding's gradients are added up in any order
    for a, p in zip(got[1:], list(m.parameters())[1:]):
        assert torch.equal(a, p.grad)


@GPU
def test_hip_token_after_a_window_of_one_step():
    """One token without gradients overwrites a one-step window's gates."""
    m = model("hip", vocab=60, hidden=40).cuda()
    x, y = batch(1, 4, 60, device="cuda")
    scores, _ = m(x, m.state_init(4))
    loss = trainer.nll_loss(scores, y)
    with torch.no_grad():
        m(x, m.state_init(4))
    with pytest.raises(RuntimeError, match="another forward pass"):
        loss.backward()


@GPU
def test_hip_layer_has_no_second_derivative():
    m = model("hip", vocab=60, hidden=40, layers=1).cuda()
    x, _ = batch(5, 3, 60, device="cuda")
    m(x, m.state_init(3))
    hm, layer = m._hip_model, m.rnns[0]
    cur = torch.randn(5, 3, 40, device="cuda").bfloat16().requires_grad_()
    out, _, _ = hm._glr_layer(cur, torch.zeros(3, 40, device="cuda"), layer,
                              hm.layers[0])
    (d,) = torch.autograd.grad(out.float().square().sum(), cur,
                               create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable"):
        d.float().sum().backward()


@GPU
@pytest.mark.parametrize("T", [129, 400])
def test_hip_a_wait_that_ends_is_told(T):
    """No look at all is allowed: every tile but the first gives up. The
    kernels end, states are NaN, and check_aborts raises."""
    from zaremba_amd import _C
    e = _C.ext()
    x, y = batch(T, 3, 60, device="cuda")
    m = model("hip", vocab=60, hidden=40).cuda()
    scores, states = m(x, m.state_init(3))
    trainer.nll_loss(scores, y).backward()
    m._hip_model.check_aborts()
    m = model("hip", vocab=60, hidden=40, layers=1).cuda()
    e.set_glr_polls(0)
    try:
        with torch.no_grad():
            short, _ = m(x[:128], m.state_init(3))
            m._hip_model.check_aborts()      # one tile waits for nobody
            scores, states = m(x, m.state_init(3))
        torch.cuda.synchronize()
    finally:
        e.set_glr_polls(1 << 22)
    assert bool(torch.isnan(states[0][1]).all())
    scores = scores.view(T, 3, -1)
    assert not torch.isnan(scores[:128]).any()
    assert bool(torch.isnan(scores[128:]).all())
    with pytest.raises(RuntimeError, match="gave up"):
        m._hip_model.check_aborts()
    # in the backward pass alone
    m = model("hip", vocab=60, hidden=40, layers=1).cuda()
    scores, _ = m(x, m.state_init(3))
    m._hip_model.check_aborts()
    e.set_glr_polls(0)
    try:
        trainer.nll_loss(scores, y).backward()
        torch.cuda.synchronize()
    finally:
        e.set_glr_polls(1 << 22)
    assert bool(torch.isnan(m.rnns[0].W_x.grad).any())
    with pytest.raises(RuntimeError, match="gave up"):
        m._hip_model.check_aborts()


@GPU
def test_gave_up_is_checked():
    from zaremba_amd import _C
    e = _C.ext()
    gates = torch.zeros(4, 3, 8, device="cuda")
    for bad in (torch.zeros(1, device="cuda"),
                torch.zeros(2, dtype=torch.int32, device="cuda"),
                torch.zeros(1, dtype=torch.int32)):
        with pytest.raises(RuntimeError, match="gave_up"):
            e.glr_forward(gates, None, None, False, None, bad)
    with pytest.raises(RuntimeError, match="set_glr_polls"):
        e.set_glr_polls(-1)


@GPU
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("cell", ["glr", "lstm"])
def test_hip_shadows_after_adamw_are_those_of_the_masters(cell, bits):
    """What a step leaves (copies, transposes, packs, folded biases) against
    what the masters give, tensor by tensor and in the next scores."""
    torch.manual_seed(0)
    m = Model(203, 72, 2, 0.0, 0.1, engine="hip", cell=cell).cuda()
    opt = AdamW(m.parameters(), bits=bits)
    for step in range(3):
        x, y = batch(11, 4, 203, seed=step, device="cuda")
        m.zero_grad(set_to_none=True)
        scores, _ = m(x, m.state_init(4))
        trainer.nll_loss(scores, y).backward()
        trainer.adamw_step(m, opt, 1e-2, 0.5)
    hm = m._hip_model
    assert hm._shadows_fresh

    def shadows():
        out = {"emb": hm.emb_W, "fc": hm.fc.W, "fcT": hm.fc.WT}
        for k, rt in enumerate(hm.layers):
            for name in ("Wx", "WxT") + (
                    ("Wh", "WhT", "WhP", "WhTP", "bias_sum")
                    if cell == "lstm" else ()):
                out[f"{name}{k}"] = getattr(rt, name)
        return {name: t.clone() for name, t in out.items()}

    def forward():
        with torch.no_grad():
            return m(x, m.state_init(4))[0].clone()

    left, a = shadows(), forward()
    hm.refresh_shadows()
    for name, t in shadows().items():
        assert torch.equal(left[name], t), name
    assert torch.equal(a, forward())
    # the update was not lost on the way: a plain copy of the new masters
    assert torch.equal(left["emb"], m.embed.W.detach().bfloat16())
    assert torch.equal(left["Wx1"], m.rnns[1].W_x.detach().bfloat16())


@GPU
@pytest.mark.parametrize("T,B,H", [(4099, 1, 72), (2048, 5, 136)])
def test_hip_model_follows_eager_over_a_long_text(monkeypatch, T, B, H):
    """Scores, states and gradients of a window that is a chain of tiles.

    A weight's gradient is the sum of what the rows (tokens) add to it. Their
    signs differ and their roundings are alike (the probabilities of all rows
    are near 1 / 203, and are rounded alike), so that the sum may be off by
    far more than GRADS of itself. Here the gate gradients are held to GRADS
    row by row, and the sums to what the rows that went into them give: a
    matrix instruction adds 32 rows to a float32 sum, a column sum 64, with
    2^-24 of the sum at each addition: under (64 + T B / 32) 2^-24 of the
    terms' magnitudes."""
    eager = model(vocab=203, hidden=H).cuda()
    hip = model("hip", vocab=203, hidden=H).cuda()
    hip.load_state_dict(eager.state_dict())
    x, y = batch(T, B, 203, device="cuda")
    layer, gates, inputs = F_ref.glr_layer, [], []

    def recorded(g, c0):
        g.retain_grad()
        gates.append(g)
        return layer(g, c0)

    def kept(cur, *rest):
        inputs.append(cur.detach().clone())
        return hip_layer(cur, *rest)

    hm = hip.hip()
    hip_layer = hm._glr_layer
    monkeypatch.setattr(hm, "_glr_layer", kept)
    out = []
    for m in (eager, hip):
        with monkeypatch.context() as patch:
            if m is eager:
                patch.setattr(F_ref, "glr_layer", recorded)
            scores, states = m(x, m.state_init(B))
        F_ref.nll_loss(scores, y).backward()
        out.append((scores, states))
    (s0, st0), (s1, st1) = out
    hm.check_aborts()
    assert rel(s1, s0) < SCORES
    for (_, c0), (_, c1) in zip(st0, st1):
        assert rel(c1, c0) < SCORES
    bound = (64 + T * B / 32) * 2.0 ** -24
    for k, rt in enumerate(hm.layers):
        d = rt.ws.dG.view(T * B, -1).double()
        assert rel(d, gates[k].grad.view(T * B, -1)) < GRADS, k
        xs = inputs[k].view(T * B, -1).double()
        for got, want, size in (
                (hip.rnns[k].b_x, d.sum(0), d.abs().sum(0)),
                (hip.rnns[k].W_x, d.t() @ xs, d.t().abs() @ xs.abs())):
            off = (got.grad.double() - want).abs()
            assert bool((off <= bound * size).all()), k


@GPU
@pytest.mark.parametrize("cell", ["glr", "lstm"])
def test_hip_side_stream_reads_what_is_freed(monkeypatch, cell):
    """The projection's weight gradient on a side stream, while the main one
    goes on to allocate: its inputs are not handed out again before."""
    def grads(side):
        monkeypatch.setenv("ZAREMBA_AMD_SIDE_STREAM", side)
        torch.manual_seed(0)
        m = Model(503, 200, 1, 0.0, 0.1, engine="hip", cell=cell).cuda()
        out = []
        for seed in range(4):
            x, y = batch(35, 20, 503, seed=seed, device="cuda")
            m.zero_grad()
            scores, states = m(x, m.state_init(20))
            loss = trainer.nll_loss(scores, y)
            del scores, states
            loss.backward()
            rooms = [torch.full((35 * 20, k), 1e30, device="cuda")
                     for k in (100, 200, 503, 503)]
            torch.cuda.synchronize()
            out.append([m.fc.W.grad.clone(), m.rnns[0].W_x.grad.clone()])
            del rooms
            m._hip_model.side_events.clear()
        return out

    assert all(torch.equal(a, b) for xs, ys in zip(grads("0"), grads("1"))
               for a, b in zip(xs, ys))
