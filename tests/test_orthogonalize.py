"""ops.orthogonalize and train.FlatMuon against the iteration in 64 bits: shapes, types, views, what they refuse, the optimizer's step."""
import math

import pytest
import torch

gpu = pytest.mark.gpu
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
COEFFS = (3.4445, -4.7750, 2.0315)


def iterate(g, steps=5, coeffs=COEFFS, eps=1e-7):
    """The definition in 64 bits, and how far an fp32-class computation may be off (Frobenius).  One step's products and roundings are off by at most
    (4 + K) w of the result's size in every singular direction (w = 2^-22: two fp16 planes; K = the sums' length enters by its square root: the roundings
    of a sum are independent), and what is off grows by at most p' (its largest derivative on the spectrum's range) in each later step.  The planes end at
    fp16's smallest step: an entry of X is off by up to 2^-25 / 2^14, so a gradient far below eps loses its small entries."""
    x = g.detach().cpu().double()
    flip = x.shape[0] > x.shape[1]
    x = x.T if flip else x
    x = x / (x.norm() + eps)
    rows = [coeffs] * steps if isinstance(coeffs[0], float) else list(coeffs)
    off, w = math.sqrt(g.numel()) * 2.0 ** -39, 2.0 ** -22
    for a, b, c in rows:
        aa = x @ x.T
        size = x.norm().item() * (abs(a) + abs(b) + abs(c))
        y = a * x + (b * aa + c * aa @ aa) @ x
        off = off * a + w * (4 + math.sqrt(max(x.shape))) * size
        x = y
    return (x.T if flip else x), off


def grads(shapes, t="fp32", seed=0, size=1e-3, noise=0.3, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    out = []
    for m, n in shapes:
        r = max(1, min(m, n) // 8)
        out.append(((torch.randn(m, r, generator=g) @ torch.randn(r, n, generator=g) / r ** 0.5 + noise * torch.randn(m, n, generator=g)) * size).to(TYPES[t]).to(device))
    return out


def check(got, mats, **how):
    assert len(got) == len(mats)
    for o, g in zip(got, mats):
        want, off = iterate(g, **how)
        u = torch.finfo(g.dtype).eps / 2
        tiny = 2.0 ** -25 * math.sqrt(g.numel()) if g.dtype == torch.float16 else 0.0
        err = (o.detach().cpu().double() - want).norm().item()
        assert o.shape == g.shape and o.dtype == g.dtype
        assert err <= off + u * want.norm().item() + tiny, (tuple(g.shape), err, off, want.norm().item())
        # and no worse than an fp32 computation would be by much: 2e-5 of the result and its rounding
        if want.norm() > 1e-3:
            assert err <= (2e-5 + u) * want.norm().item() + tiny, (tuple(g.shape), err / max(want.norm().item(), 1e-300))


def test_iterate_moves_singular_values_to_one():
    g = grads([(20, 50)], device="cpu")[0]
    s = torch.linalg.svdvals(iterate(g)[0])
    assert 0.3 < s.min() and s.max() < 1.3


@pytest.mark.parametrize("args, kw, says", [
    ([torch.zeros(4)], {}, "matrices"), ([torch.zeros(4, 4).double()], {}, "matrices"), ([torch.zeros(2, 2, 2)], {}, "matrices"),
    ([torch.zeros(4, 4)], dict(steps=0), "steps"), ([torch.zeros(4, 4)], dict(steps=65), "steps"), ([torch.zeros(4, 4)], dict(coeffs=(1.0, 2.0)), "three"),
    ([torch.zeros(4, 4)], dict(coeffs=(1.0, 2.0, float("nan"))), "finite"), ([torch.zeros(4, 4)], dict(steps=2, coeffs=[COEFFS] * 3), "three for each"),
    ([torch.zeros(4, 4)], dict(coeffs=(50.0, 1.0, 1.0)), "without bound"), ([torch.zeros(4, 4)], dict(eps=-1.0), "eps"),
    ([torch.zeros(4, 4)], dict(eps=float("nan")), "eps"), ([torch.zeros(4, 4)], dict(out=[]), "out must"),
    ([torch.zeros(4, 4)], dict(out=[torch.zeros(4, 5)]), "out must"), ([torch.zeros(4, 4)], dict(out=[torch.zeros(4, 4).half()]), "out must"),
    ([torch.zeros(4, 4)], dict(out=[torch.zeros(4, 4).t()[:, ::2].repeat(1, 2).t()]), "contiguous columns"), ([torch.zeros(4, 4)], {}, "device tensors"),
    ([torch.empty(1, 1).expand(40000, 40000)], {}, "smaller side")])
def test_refusals(args, kw, says):
    from craft_amd import ops
    from craft_amd.hip import CraftHipError
    with pytest.raises(CraftHipError, match=says):
        ops.orthogonalize(args, **kw)


def test_entry_points_check_their_arguments():
    import ctypes

    from craft_amd import hip
    lib, buf = hip.load(), 4096
    ARG, UNSUPPORTED = 10001, 10003
    co = (ctypes.c_float * 3)(*COEFFS)

    def run(job=(buf, 8, buf, 8, 8, 8), n=1, coeffs=co, steps=1, eps=1e-7, s=(1.0, 1.0, 1.0), dt=0, ws=buf, nbytes=1 << 20):
        return lib.craft_orthogonalize((ctypes.c_long * 6)(*job), n, coeffs, steps, eps, *s, dt, ws, nbytes, None)
    assert run(n=0) == ARG and run(n=61) == ARG and run(steps=0) == ARG and run(coeffs=None) == ARG and run(eps=-1.0) == ARG and run(dt=3) == ARG
    assert run(s=(0.0, 1.0, 1.0)) == ARG and run(ws=None) == ARG and run(ws=buf + 16) == ARG and run(nbytes=8192 + 2048 + 20 * 4096 - 1) == ARG
    assert run((0, 8, buf, 8, 8, 8)) == ARG and run((buf, 8, buf, 7, 8, 8)) == ARG and run((buf, 8, buf, 8, 0, 8)) == ARG
    assert run((buf, 40000, buf, 40000, 40000, 40000)) == UNSUPPORTED
    seg = (ctypes.c_long * 2)(0, 8)
    assert lib.craft_muon_momentum(None, buf, buf, seg, 1, 0.9, 1, buf, None) == ARG and lib.craft_muon_momentum(buf, buf, buf, seg, 1, 1.0, 1, buf, None) == ARG
    assert lib.craft_muon_momentum(buf, buf, buf, (ctypes.c_long * 2)(-1, 8), 1, 0.9, 1, buf, None) == ARG
    assert lib.craft_muon_apply(buf, buf, seg, None, 1, 0.1, 0.0, buf, None) == ARG


@gpu
@pytest.mark.parametrize("shapes", [[(1, 1)], [(1, 70)], [(70, 1)], [(64, 64)], [(65, 64)], [(16, 300)], [(300, 16)], [(127, 129)], [(200, 500), (500, 200)],
                                    [(64, 147), (126, 600), (2, 3), (15, 15), (256, 324), (96, 64), (1, 5)], [(20 + i, 40 + 3 * i) for i in range(66)]],
                         ids=lambda s: f"{len(s)}of{s[0][0]}x{s[0][1]}")
@pytest.mark.parametrize("t", list(TYPES))
def test_against_64_bits(device, t, shapes):
    from craft_amd import ops
    mats = grads(shapes, t)
    check(ops.orthogonalize(mats), mats)


@gpu
def test_large(device):
    from craft_amd import ops
    for shape in ((700, 2300), (1024, 1024), (1100, 640), (257, 257), (300, 5000), (256, 9000)):
        mats = grads([shape])
        check(ops.orthogonalize(mats), mats)
    mats = grads([(300, 700), (64, 64), (1000, 520), (100, 3000), (400, 400)])
    check(ops.orthogonalize(mats), mats)


@gpu
def test_steps_coefficients_and_sizes(device):
    """One and many steps, other polynomials, one for each step; gradients far from unit size; the norm counts from 1e-7 on."""
    from craft_amd import ops
    for steps, coeffs in ((1, COEFFS), (2, COEFFS), (8, (1.5, -0.5, 0.0)), (3, [(4.0, -6.0, 2.5), (3.0, -3.5, 1.4), (2.0, -1.5, 0.5)])):
        mats = grads([(60, 200), (130, 70)])
        check(ops.orthogonalize(mats, steps=steps, coeffs=coeffs), mats, steps=steps, coeffs=coeffs)
    for size in (1e-20, 1e-7, 1e6, 1e15):
        mats = grads([(60, 200)], size=size)
        check(ops.orthogonalize(mats), mats)
    mats = grads([(60, 200)])
    check(ops.orthogonalize(mats, eps=0.0), mats, eps=0.0)


@gpu
def test_zero_and_nan(device):
    """A matrix of zeros stays one; one that holds a NaN or an infinity spoils itself only."""
    from craft_amd import ops
    mats = grads([(40, 90), (40, 90), (40, 90), (40, 90)])
    mats[0].zero_()
    mats[1][3, 4] = math.nan
    mats[2][0, 0] = math.inf
    out = ops.orthogonalize(mats)
    assert not out[0].any() and out[1].isnan().all() and not out[2].isfinite().any()
    check(out[3:], mats[3:])
    one = torch.zeros(30, 50, device="cuda")
    one[7, 9] = 5.0                                                        # rank one: the one entry follows the scalar polynomial
    check(ops.orthogonalize([one]), [one])


@gpu
def test_views_out_streams_and_graphs(device):
    from craft_amd import ops
    g = grads([(90, 130)])[0]
    views = [g.t(), g[::2], g[:, ::3], g[5:50, 7:77]]
    check(ops.orthogonalize(views), views)
    flat = torch.zeros(100 + 90 * 130, device="cuda")
    out = flat[100:].view(90, 130)
    assert ops.orthogonalize([g], out=[out])[0].data_ptr() == out.data_ptr()
    check([out], [g])
    assert not flat[:100].any()
    wide = torch.zeros(90, 200, device="cuda")
    ops.orthogonalize([g], out=[wide[:, 30:160]])
    check([wide[:, 30:160]], [g])
    assert not wide[:, :30].any() and not wide[:, 160:].any()
    same = g.clone()
    assert torch.equal(ops.orthogonalize([same], out=[same])[0], out)      # in place
    assert ops.orthogonalize([]) == [] and ops.orthogonalize([torch.zeros(0, 5, device="cuda")])[0].shape == (0, 5)
    mixed = grads([(50, 60)], "fp16") + grads([(50, 60)], "fp32") + grads([(70, 20)], "bf16")
    check(ops.orthogonalize(mixed), mixed)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.orthogonalize([g])[0]
    side.synchronize()
    assert torch.equal(other, out)
    mats = grads([(64, 300), (200, 90)])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = ops.orthogonalize(mats)
    for seed in range(4):
        for a, b in zip(mats, grads([(64, 300), (200, 90)], seed=seed)):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(res, ops.orthogonalize(mats)))


# ---------------------------------------------------------------------------------------------------------------- the optimizer
def net(seed=0, device="cpu"):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Conv2d(16, 24, 3), torch.nn.BatchNorm2d(24), torch.nn.Conv2d(24, 8, 3, bias=False), torch.nn.Linear(40, 100),
                               torch.nn.Linear(100, 20)).to(device)


def test_muon_partition_and_state():
    """Which parameters are matrices, and that states go round and refuse the other optimizer's."""
    from craft_amd.train import FlatAdamW, FlatMuon
    n = net()
    opt = FlatMuon(n.parameters(), lr=1e-2)
    names = [k for k, _ in n.named_parameters()]
    assert [names[i] for i in opt.matrix_index] == ["0.weight", "3.weight", "4.weight"]      # (the 8-row convolution is below matrix_min)
    covered = torch.zeros(opt.numel, dtype=torch.int32)
    for a, b in opt.adam_segments:
        covered[a:b] += 1
    for off, m in opt._segs:
        covered[off:off + m] += 1
    assert int(covered.max()) == 1
    for off, p in zip(opt.offsets, opt.params):
        assert bool((covered[off:off + p.numel()] == 1).all())
    opt.exp_avg.copy_(torch.randn(opt.numel))
    sd = opt.state_dict()
    assert set(sd["state"][0]) == {"step", "momentum_buffer"} and set(sd["state"][1]) == {"step", "exp_avg", "exp_avg_sq"}
    again = FlatMuon(net(1).parameters())
    again.load_state_dict(sd)
    for off, p in zip(opt.offsets, opt.params):
        assert torch.equal(again.exp_avg[off:off + p.numel()], opt.exp_avg[off:off + p.numel()])
    assert again.lr == 1e-2
    with pytest.raises(ValueError, match="another optimizer"):
        FlatAdamW(net().parameters()).load_state_dict(sd)
    with pytest.raises(ValueError, match="another optimizer"):
        again.load_state_dict(FlatAdamW(net().parameters()).state_dict())
    with pytest.raises(ValueError, match="momentum"):
        FlatMuon(net().parameters(), momentum=1.0)
    assert FlatMuon(net().parameters(), matrix_min=1000).matrix_index == []


def test_optimizer_choice():
    from craft_amd.train import FlatAdamW, FlatMuon, fetch_optimizer
    from craft_amd.train_main import parse
    m = torch.nn.Linear(32, 32)
    assert type(fetch_optimizer(m, 1e-3, 1e-4, 1e-8, 10)[0]) is FlatAdamW and type(fetch_optimizer(m, 1e-3, 1e-4, 1e-8, 10, "muon")[0]) is FlatMuon
    with pytest.raises(ValueError, match="one of adamw, muon"):
        fetch_optimizer(m, 1e-3, 1e-4, 1e-8, 10, "sgd")
    assert parse(["--stage", "chairs"]).optimizer == "adamw" and parse(["--stage", "chairs", "--optimizer", "muon"]).optimizer == "muon"


@gpu
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_steps_against_64_bits(device, nesterov):
    """Three steps with clipping, weight decay and a loss scale, matrices by the definition in 64 bits, the rest by torch's AdamW; then a step that an
    overflow skips.  A matrix' step is lr s O with entries of O off by at most 2e-5 of its rms in the mean (see check): summed over three steps."""
    from craft_amd.train import FlatMuon
    lr, wd, mu, clip, scale = 3e-2, 1e-2, 0.9, 1.0, 64.0
    n, ref = net(3, "cuda"), net(3, "cuda").double()
    opt = FlatMuon(n.parameters(), lr=lr, weight_decay=wd, momentum=mu, nesterov=nesterov)
    opt.set_loss_scale(scale)
    rp = list(ref.parameters())
    rest = [i for i in range(len(rp)) if i not in opt.matrix_index]
    adam = torch.optim.AdamW([rp[i] for i in rest], lr=lr, weight_decay=wd, eps=1e-8)
    buf = {i: torch.zeros_like(rp[i]) for i in opt.matrix_index}
    for step in range(3):
        g = torch.Generator().manual_seed(step)
        gs = [torch.randn(p.shape, generator=g).cuda() for p in rp]
        for p, d in zip(opt.params, gs):
            p.grad.copy_(d * scale)
        opt.step(max_norm=clip)
        f = min(1.0, clip / (math.sqrt(sum(d.double().square().sum().item() for d in gs)) + 1e-6))
        for p, d in zip(rp, gs):
            p.grad = d.double() * f
        adam.step()
        for i in opt.matrix_index:
            buf[i] = mu * buf[i] + rp[i].grad
            u = rp[i].grad + mu * buf[i] if nesterov else buf[i]
            o, _ = iterate(u.view(u.shape[0], -1))
            with torch.no_grad():
                rp[i].mul_(1 - lr * wd).sub_(lr * 0.2 * math.sqrt(max(o.shape)) * o.cuda().view_as(rp[i]))
    for i, (p, r) in enumerate(zip(opt.params, rp)):
        off = (p.double() - r).norm().item()
        assert off <= (2e-5 * lr * 0.2 * 3 + 6e-7) * math.sqrt(p.numel()) + 1e-6 * r.norm().item(), (i, off)
    assert opt.step_count == 3
    before, m = opt.flat.clone(), opt.exp_avg.clone()
    opt.flat_grad[5] = math.inf
    opt.step(max_norm=clip)
    assert torch.equal(before, opt.flat) and torch.equal(m, opt.exp_avg) and opt.step_count == 3


@gpu
def test_trainer_with_muon(device):
    """Trainer(optimizer="muon") moves the model's matrices by the update's rms and everything else by AdamW, and its checkpoint restores."""
    from craft_amd import CRAFT, default_args
    from craft_amd.synth import synth_pair, synth_state_dict
    from craft_amd.train import FlatMuon, Trainer
    model = CRAFT(default_args())
    model.load_state_dict(synth_state_dict(model.state_dict(), seed=5), strict=True)
    model = model.to("cuda")
    tr = Trainer(model, lr=1e-3, wdecay=0.0, iters=2, num_steps=100, optimizer="muon")
    opt = tr.optimizer
    assert isinstance(opt, FlatMuon) and len(opt.matrix_index) == 53
    im1, im2, flow = synth_pair(1, 128, 160, seed=0)
    before, lr = opt.flat.clone(), tr.scheduler.get_last_lr()[0]
    m = tr.step(im1, im2, flow, torch.ones(1, 128, 160))
    assert math.isfinite(m["loss"]) and opt.step_count == 1
    for i in opt.matrix_index:
        off, n = opt.offsets[i], opt.params[i].numel()
        d = (opt.flat[off:off + n] - before[off:off + n]).double().square().mean().sqrt().item()
        assert d <= 1.3 * 0.2 * lr, (i, d, lr)                             # singular values up to 1.2
    sd = opt.state_dict()
    opt.load_state_dict(sd)
    assert len(sd["state"]) == len(opt.params) - len(opt.unused_index)


def test_results_in_one_place_are_refused():
    from craft_amd import ops
    from craft_amd.hip import CraftHipError
    a, b = torch.zeros(4, 4), torch.zeros(4, 4)
    with pytest.raises(CraftHipError, match="two results"):
        ops.orthogonalize([a, b], out=[a, a])
    with pytest.raises(CraftHipError, match="two results"):
        ops.orthogonalize([a, a], out=[a, a])
    with pytest.raises(CraftHipError, match="another matrix"):
        ops.orthogonalize([a, b], out=[b, a])
    with pytest.raises(CraftHipError, match="device tensors"):             # (the same matrix twice, results of their own: fine)
        ops.orthogonalize([a, a])


@pytest.mark.parametrize("over", [dict(pos_bias_radius=9), dict(pos_bias_radius=7), dict(use_setrans=False, position_and_content=True),
                                  dict(use_setrans=False)])
def test_position_tables_are_adamws(over):
    """Tables of 16 rows and columns or more (a radius of 9: 19 x 19; relative positions: 319 x 128) are no matrices, whatever their shape."""
    from craft_amd import CRAFT, default_args
    from craft_amd.train import fetch_optimizer
    model = CRAFT(default_args(**over))
    opt, _ = fetch_optimizer(model, 1e-3, 1e-4, 1e-8, 10, "muon")
    names = [k for k, _ in model.named_parameters()]
    matrices = {names[i] for i in opt.matrix_index}
    tables = {k for k in names if k.endswith("pos_coder.biases") or "rel_height" in k or "rel_width" in k}
    assert tables and not tables & matrices
    shapes = {k: (p.shape[0], p.numel() // p.shape[0]) for k, p in model.named_parameters() if p.dim() >= 2}
    unused = {names[i] for i in opt.unused_index}
    assert matrices == {k for k, v in shapes.items() if min(v) >= 16} - tables - unused
    at = {names.index(k) for k in tables - unused}
    for i in at:
        assert any(a <= opt.offsets[i] and opt.offsets[i] + opt.params[i].numel() <= b for a, b in opt.adam_segments)
        assert set(opt.state_dict()["state"][i]) == {"step", "exp_avg", "exp_avg_sq"}


def test_a_state_that_does_not_fit_changes_nothing():
    """Refused before any of it is taken over: the first parameters of these nets have states that either optimizer could read."""
    from craft_amd.train import FlatAdamW, FlatMuon
    nets = lambda width: torch.nn.Sequential(torch.nn.LayerNorm(40), torch.nn.Linear(40, width))     # noqa: E731
    muon, adam = FlatMuon(nets(32).parameters(), lr=0.5), FlatAdamW(nets(32).parameters(), lr=0.25)
    wide = FlatAdamW(nets(48).parameters(), lr=0.125)
    for opt in (muon, adam, wide):
        opt.exp_avg.fill_(opt.lr)
        opt.step_count = 7
    for opt, other, says in ((adam, muon, "another optimizer"), (muon, adam, "another optimizer"), (adam, wide, "the parameter")):
        fresh = type(opt)(nets(32).parameters(), lr=3.0)
        with pytest.raises(ValueError, match=says):
            fresh.load_state_dict(other.state_dict())
        assert not fresh.exp_avg.any() and not fresh.exp_avg_sq.any() and fresh.step_count == 0 and fresh.lr == 3.0


@gpu
@pytest.mark.parametrize("size", [1e-44, 1e-40, 1e-36, 1e-30, 1e30, 1e37])
@pytest.mark.parametrize("shape", [(60, 200), (300, 280)])
def test_norms_at_the_ends_of_fp32(device, size, shape):
    """Without an eps a matrix of any size that is not zero has a direction; the factor to it does not fit fp32, nor does the norm of the largest."""
    from craft_amd import ops
    mats = [(g.double() * size).float() for g in grads([shape], size=1.0)]
    assert mats[0].any() and mats[0].isfinite().all()
    check(ops.orthogonalize(mats, eps=0.0), mats, eps=0.0)
    assert ops.orthogonalize([torch.zeros(5, 9, device="cuda")], eps=0.0)[0].isnan().all()
