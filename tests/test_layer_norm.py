"""ops.layer_norm / autograd.layer_norm against the formula in 64 bits: types, widths, strides, what they refuse."""
import pytest
import torch

gpu = pytest.mark.gpu
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def norm64(x, w, b, dy, eps=1e-5):
    """(y, dx, dw, db) and their tolerances: the final rounding (u of each output's type), the fp32 sums (as many roundings as they have terms, of the
    terms' size) and a few roundings of each step's own size."""
    e = 2.0 ** -24
    xd, dyd = x.detach().cpu().double(), dy.cpu().double()
    C, R = x.shape[-1], x.shape[0]
    wd = torch.ones(C, dtype=torch.float64) if w is None else w.detach().cpu().double()
    bd = torch.zeros(C, dtype=torch.float64) if b is None else b.detach().cpu().double()
    wt = torch.float32 if w is None and b is None else (w if w is not None else b).dtype
    mean = xd.mean(-1, keepdim=True)
    var = (xd - mean).square().mean(-1, keepdim=True)
    rstd = (var + eps).rsqrt()
    xn = (xd - mean) * rstd
    y = xn * wd + bd
    # the mean is off by C roundings of the mean magnitude; a sum over 16 .. 1024 threads is far shorter than that, but the bound holds for any order
    em = (C + 2) * e * xd.abs().mean(-1, keepdim=True)
    en = rstd * (em + e * xd.abs()) + xn.abs() * ((C + 8) * e + rstd ** 2 * em ** 2)         # of xn (var: C roundings of itself, and the mean's error squared)
    u = lambda t: torch.finfo(t).eps / 2                                                      # noqa: E731
    ty = wd.abs() * en + u(x.dtype) * y.abs() + 4 * e * (y.abs() + bd.abs())
    g = dyd * wd
    m0, m1 = g.mean(-1, keepdim=True), (g * xn).mean(-1, keepdim=True)
    dx = rstd * (g - m0 - xn * m1)
    e0 = (C + 4) * e * g.abs().mean(-1, keepdim=True)
    e1 = (C + 4) * e * (g * xn).abs().mean(-1, keepdim=True) + (g.abs() * en).mean(-1, keepdim=True)
    tx = rstd * (e0 + xn.abs() * e1 + en * m1.abs() + 8 * e * (g.abs() + m0.abs() + (xn * m1).abs())) + dx.abs() * (C + 8) * e + u(x.dtype) * dx.abs()
    dw, db = (dyd * xn).sum(0), dyd.sum(0)
    tw = (dyd.abs() * en).sum(0) + (R + 4) * e * (dyd * xn).abs().sum(0) + u(wt) * dw.abs()
    tb = (R + 4) * e * dyd.abs().sum(0) + u(wt) * db.abs()
    return (y, dx, dw, db), (ty, tx, tw, tb)


def check(got, want, tol):
    for g, r, e, name in zip(got, want, tol, ("y", "dx", "dw", "db")):
        if g is None:
            continue
        off = (g.detach().cpu().double() - r).abs()
        assert g.shape == r.shape and torch.isfinite(off).all(), name
        # (fp16's smallest steps: an absolute half of 2^-24)
        worst = (off / (e + (2.0 ** -25 if g.dtype == torch.float16 else 1e-30))).max().item()
        assert worst <= 1.0, f"{name}: {worst:.2f} times the bound, at most {off.max().item():.3g} off"


def make(t, rows, C, seed=0, offset=0.5, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)                            # noqa: E731
    return ((n(rows, C) * (0.5 + n(rows, 1).abs()) + offset * n(rows, 1)).to(TYPES[t]).to(device), (1 + 0.2 * n(C)).to(device), (0.1 * n(C)).to(device),
            n(rows, C).to(TYPES[t]).to(device))


def test_formula_is_autograds():
    x, w, b, dy = make("fp32", 7, 33, device="cpu")
    want, _ = norm64(x, w, b, dy)
    xd, wd, bd = (v.double().requires_grad_() for v in (x, w, b))
    y = torch.nn.functional.layer_norm(xd, (33,), wd, bd, 1e-5)
    for a, r in zip((y, *torch.autograd.grad(y, (xd, wd, bd), dy.double())), want):
        assert torch.allclose(a, r, rtol=1e-11, atol=1e-11)


@pytest.mark.parametrize("x, w, b, eps, says", [
    (torch.zeros(2, 4, dtype=torch.float64), None, None, 1e-5, "fp32, fp16 or bf16"),
    (torch.zeros(2, 4, dtype=torch.int32), None, None, 1e-5, "fp32, fp16 or bf16"),
    (torch.zeros(2, 0), None, None, 1e-5, "last axis"), (torch.zeros(2, 16385), None, None, 1e-5, "last axis"), (torch.zeros(()), None, None, 1e-5, "last axis"),
    (torch.zeros(2, 4), torch.zeros(3), None, 1e-5, "weight must"), (torch.zeros(2, 4), torch.zeros(4).half(), None, 1e-5, "weight must"),
    (torch.zeros(2, 4), None, torch.zeros(1, 4), 1e-5, "bias must"), (torch.zeros(2, 4).half(), torch.zeros(4), torch.zeros(4).half(), 1e-5, "one type"),
    (torch.zeros(2, 4).half(), torch.zeros(4).bfloat16(), None, 1e-5, "weight must"),
    (torch.zeros(2, 4), None, None, -1.0, "eps"), (torch.zeros(2, 4), None, None, float("nan"), "eps"), (torch.zeros(2, 4), None, None, 1e-5, "device tensors")])
def test_refusals(x, w, b, eps, says):
    from craft_amd import autograd, ops
    from craft_amd.hip import CraftHipError
    for f in (ops.layer_norm, autograd.layer_norm):
        with pytest.raises(CraftHipError, match=says):
            f(x, w, b, eps)


def test_entry_points_check_their_arguments():
    from craft_amd import hip
    lib, buf = hip.load(), 4096
    fwd = lambda x=buf, ldx=8, rows=2, C=8, eps=1e-5, dt=0, wdt=0, y=buf, ldy=8, mean=None, rstd=None: lib.craft_layer_norm_fwd(x, ldx, None, None, rows, C, eps, dt, wdt, y, ldy, mean, rstd, None)  # noqa: E731
    ARG, ALIGN, UNSUPPORTED = 10001, 10002, 10003
    assert fwd(rows=0) == ARG and fwd(C=0) == ARG and fwd(C=16385, ldy=16385) == UNSUPPORTED and fwd(eps=-1.0) == ARG and fwd(eps=float("nan")) == ARG
    assert fwd(x=None) == ARG and fwd(ldx=-1) == ARG and fwd(ldy=7) == ARG and fwd(x=buf + 2) == ALIGN and fwd(x=buf + 1, dt=2, wdt=2) == ALIGN
    assert fwd(mean=buf) == ARG and fwd(dt=3) == ARG and fwd(dt=0, wdt=2) == UNSUPPORTED and fwd(dt=1, wdt=2) == UNSUPPORTED
    bwd = lambda dx=buf, dw=buf, ws=buf, blocks=4, mean=buf, lddx=8, lddy=8: lib.craft_layer_norm_bwd(buf, 8, buf, lddy, None, mean, buf, 2, 8, 0, 0, dx, lddx, dw, None, ws, blocks, None)  # noqa: E731
    assert bwd(ws=None) == ARG and bwd(blocks=0) == ARG and bwd(mean=None) == ARG and bwd(lddx=7) == ARG and bwd(lddy=-8) == ARG


@gpu
@pytest.mark.parametrize("t, wt", [("fp32", "fp32"), ("fp16", "fp16"), ("fp16", "fp32"), ("bf16", "bf16"), ("bf16", "fp32")])
@pytest.mark.parametrize("rows, C", [(1, 1), (3, 2), (1, 7), (70, 46), (5, 127), (129, 129), (9, 256), (300, 257), (33, 1000), (17, 1027), (7, 2049), (3, 4096), (4, 4100),
                                     (2, 8193), (2, 16384), (2500, 24)])
def test_against_64_bits(device, t, wt, rows, C):
    from craft_amd import autograd, ops
    x, w, b, dy = make(t, rows, C)
    w, b = w.to(TYPES[wt]), b.to(TYPES[wt])
    want, tol = norm64(x, w, b, dy)
    check([ops.layer_norm(x, w, b)], want, tol)
    x, w, b = (v.requires_grad_() for v in (x, w, b))
    y = autograd.layer_norm(x, w, b)
    got = torch.autograd.grad(y, (x, w, b), dy)
    check([y, *got], want, tol)
    assert got[0].dtype == x.dtype and got[1].dtype == w.dtype and got[2].dtype == b.dtype


@gpu
def test_without_weights_and_some_gradients(device):
    from craft_amd import autograd
    for keep in ((True, False), (False, True), (False, False)):
        x, w, b, dy = make("bf16", 50, 200)
        w, b = (v.to(torch.bfloat16).requires_grad_() if k else None for v, k in zip((w, b), keep))
        want, tol = norm64(x, w, b, dy)
        x.requires_grad_()
        y = autograd.layer_norm(x, w, b)
        leaves = [v for v in (x, w, b) if v is not None]
        got = dict(zip(map(id, leaves), torch.autograd.grad(y, leaves, dy, retain_graph=True)))
        check([y, got[id(x)], got.get(id(w)) if w is not None else None, got.get(id(b)) if b is not None else None], want, tol)
        for v, r, e in ((w, want[2], tol[2]), (b, want[3], tol[3])):       # a weight's gradient alone
            if v is not None:
                check([torch.autograd.grad(y, v, dy, retain_graph=True)[0]], [r], [e])


@gpu
def test_large_offset_and_constant_rows(device):
    """Rows far from zero keep their spread (the squares are summed about the mean), rows of one value give the bias."""
    from craft_amd import ops
    x, w, b, dy = make("fp32", 40, 300, offset=300.0)
    want, tol = norm64(x, w, b, dy)
    check([ops.layer_norm(x, w, b)], want, tol)
    y = ops.layer_norm(torch.full((3, 500), 7.25, device="cuda", dtype=torch.float16), None, b.new_full((500,), 0.5).half())
    assert torch.equal(y, torch.full_like(y, 0.5))


@gpu
def test_views_out_and_empty(device):
    from craft_amd import autograd, ops
    big = torch.randn(6, 40, 100, generator=torch.Generator().manual_seed(2)).half().cuda()
    for x in (big[:, :, 3:80], big[1], big.transpose(0, 1), big[:, ::2, 1:], big[0, :, :1], big[:, 5, 7:], big[2, 3]):
        flat = x.reshape(-1, x.shape[-1])
        want, tol = norm64(flat, None, None, flat)
        check([ops.layer_norm(x).reshape(flat.shape)], want, tol)
    out = torch.zeros(40, 100, device="cuda", dtype=torch.float16)
    want, tol = norm64(big[1][:, :90], None, None, big[1][:, :90])
    ops.layer_norm(big[1][:, :90], out=out[:, 5:95])
    check([out[:, 5:95]], want, tol)
    assert not out[:, :5].any() and not out[:, 95:].any()
    same = big[1].clone()
    assert torch.equal(ops.layer_norm(same, out=same), ops.layer_norm(big[1]))
    with pytest.raises(Exception, match="out must"):
        ops.layer_norm(big[1], out=out.t()[:40, :40])
    x = torch.zeros(0, 5, device="cuda", requires_grad=True)
    w = torch.ones(5, device="cuda", requires_grad=True)
    y = autograd.layer_norm(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert y.shape == dx.shape == (0, 5) and not dw.any()
    # one gradient row for all
    x, w, b, _ = make("fp32", 30, 64)
    x.requires_grad_()
    row = torch.randn(64, device="cuda")
    want, tol = norm64(x, w, b, row.expand(30, 64))
    check([None, torch.autograd.grad(autograd.layer_norm(x, w, b), x, row.expand(30, 64))[0]], want, tol)


@gpu
def test_gradients_against_differences(device):
    """Central differences of the kernel's own forward pass: an fp32 sum of 20 x 37 products of unit size is off by at most 5e-5, which a step of 2e-2 turns
    into 3e-3 of a derivative of size 1 to 10."""
    from craft_amd import autograd
    x, w, b, dy = make("fp32", 20, 37)
    x, w, b = (v.requires_grad_() for v in (x, w, b))
    grads = torch.autograd.grad(autograd.layer_norm(x, w, b), (x, w, b), dy)
    for n, v in enumerate((x, w, b)):
        d = torch.randn(v.shape, generator=torch.Generator().manual_seed(n)).cuda()
        f = lambda s: (autograd.layer_norm(*[a.detach() + (s * d if m == n else 0) for m, a in enumerate((x, w, b))]).double() * dy.double()).sum().item()  # noqa: E731,B023
        num = (f(1e-2) - f(-1e-2)) / 2e-2
        assert abs(num - (grads[n].double() * d.double()).sum().item()) < 1e-2 * max(1.0, abs(num))


@gpu
def test_same_bits_and_captured(device):
    from craft_amd import ops
    x, w, b, _ = make("bf16", 500, 770)
    a = ops.layer_norm(x, w, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = ops.layer_norm(x, w, b)
    side.synchronize()
    assert torch.equal(a, y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, mean, rstd = ops._layer_norm(x, w, b, 1e-5, None, True)
        grads = ops.layer_norm_bwd(x, w, b.dtype, a, mean, rstd)
    for seed in range(4):
        x.copy_(make("bf16", 500, 770, seed)[0])
        graph.replay()
        torch.cuda.synchronize()
        y2, mean2, rstd2 = ops._layer_norm(x, w, b, 1e-5, None, True)
        assert torch.equal(y, y2) and all(torch.equal(p, q) for p, q in zip(grads, ops.layer_norm_bwd(x, w, b.dtype, a, mean2, rstd2)))


@pytest.mark.parametrize("change, says", [
    (dict(dy=torch.zeros(3, 4)), "dy"), (dict(dy=torch.zeros(2, 5)), "dy"), (dict(mean=torch.zeros(1)), "mean and rstd"),
    (dict(rstd=torch.zeros(2).double()), "mean and rstd"), (dict(mean=torch.zeros(4)[::2]), "mean and rstd"), (dict(weight=torch.zeros(3)), "weight must"),
    (dict(bias_type=torch.float16), "dy"), (dict(), "device tensors")])
def test_backward_refusals(change, says):
    from craft_amd import ops
    from craft_amd.hip import CraftHipError
    args = dict(x=torch.zeros(2, 4), weight=None, bias_type=None, dy=torch.zeros(2, 4), mean=torch.zeros(2), rstd=torch.zeros(2))
    args.update(change)
    with pytest.raises(CraftHipError, match=says):
        ops.layer_norm_bwd(**args)


@gpu
@pytest.mark.parametrize("rows, C", [(5, 7), (70, 46), (300, 257), (17, 1027), (600, 4100)])
def test_in_place(device, rows, C):
    from craft_amd import ops
    x = torch.randn(rows, C, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    want = ops.layer_norm(x)
    assert ops.layer_norm(x, out=x) is x and torch.equal(x, want)
    # rows that are one row in memory
    one = x[:1].expand(rows, C)
    assert torch.equal(ops.layer_norm(one), ops.layer_norm(one.contiguous()))


def norm64_deep(x, w, b, dy, eps=1e-5):
    """norm64 with the depth of the kernels' sums in place of their length, so that one lost row shows.  A row has 16, 64, 128, ... 1024 threads, the fewest
    that hold its 16-byte vectors: a thread's values, 6 steps over a wave, up to 16 waves, 4 for the quotient and differences.  A weight's gradient: the rows of
    a group of threads, the groups of a block, 16 + 16 blocks."""
    e, C, R = 2.0 ** -24, x.shape[-1], x.shape[0]
    vectors = -(-C * x.element_size() // 16)
    threads = next((n for n in (16, 64, 128, 256, 512) if vectors <= n), 1024)
    row = 16 // x.element_size() * -(-vectors // threads) + 6 + -(-threads // 64) + 4
    col = -(-R * threads // (256 * 1024)) + 1024 // threads + 32
    xd, dyd, wd, bd = (v.detach().cpu().double() for v in (x, dy, w, b))
    xd = xd.requires_grad_()
    wl, bl = wd.clone().requires_grad_(), bd.clone().requires_grad_()
    y = torch.nn.functional.layer_norm(xd, (C,), wl, bl, eps)
    dx, dw, db = torch.autograd.grad(y, (xd, wl, bl), dyd)
    y, xd = y.detach(), xd.detach()
    mean = xd.mean(-1, keepdim=True)
    rstd = ((xd - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    xn = (xd - mean) * rstd
    em = row * e * xd.abs().mean(-1, keepdim=True)
    en = rstd * (em + e * xd.abs()) + xn.abs() * (row * e + rstd ** 2 * em ** 2)
    u = lambda v: torch.finfo(v.dtype).eps / 2                             # noqa: E731
    ty = wd.abs() * en + u(x) * y.abs() + 4 * e * (y.abs() + bd.abs())
    g = dyd * wd
    m0, m1 = g.mean(-1, keepdim=True), (g * xn).mean(-1, keepdim=True)
    e0 = row * e * g.abs().mean(-1, keepdim=True)
    e1 = row * e * (g * xn).abs().mean(-1, keepdim=True) + (g.abs() * en).mean(-1, keepdim=True)
    tx = rstd * (e0 + xn.abs() * e1 + en * m1.abs() + 8 * e * (g.abs() + m0.abs() + (xn * m1).abs())) + dx.abs() * row * e + u(x) * dx.abs()
    tw = (dyd.abs() * en).sum(0) + col * e * (dyd * xn).abs().sum(0) + u(w) * dw.abs()
    tb = col * e * dyd.abs().sum(0) + u(b) * db.abs()
    return (y, dx, dw, db), (ty, tx, tw, tb), dyd * xn


# rows so many that every group of threads meets at least three (256 blocks of 1024 / TPR groups), and an odd number of them
MANY = [(50021, 24), (13001, 257), (13001, 136), (6501, 520), (3333, 1027), (1701, 2056), (901, 4100), (901, 8192), (781, 16384)]


@pytest.mark.parametrize("rows, C", [(50021, 24), (901, 4100)])
def test_many_rows_bound_shows_a_lost_row(rows, C):
    """The oracle's bounds on the weights' gradients are below what a row brings, in more than half of its columns on the average over the rows."""
    x, w, b, dy = make("bf16", rows, C, device="cpu")
    _, tol, term = norm64_deep(x, w, b, dy)
    assert (term.abs() > tol[2]).double().mean() > 0.5 and (dy.double().abs() > tol[3]).double().mean() > 0.5


@gpu
@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("rows, C", MANY)
def test_many_rows(device, t, rows, C):
    """The walk over rows: the next row's prefetch, the alternating buffers of its sums, the weights' gradients held over all of them."""
    from craft_amd import autograd, ops
    x, w, b, dy = make(t, rows, C)
    want, tol, _ = norm64_deep(x, w, b, dy)
    check([ops.layer_norm(x, w, b)], want, tol)
    x, w, b = (v.requires_grad_() for v in (x, w, b))
    y = autograd.layer_norm(x, w, b)
    check([y, *torch.autograd.grad(y, (x, w, b), dy)], want, tol)


@gpu
def test_second_derivatives_are_refused(device):
    """The backward pass has none of its own: asked for (create_graph), its results raise when they are differentiated, and are right until then."""
    from craft_amd import autograd
    x, w, b, dy = make("fp32", 20, 70)
    want, tol = norm64(x, w, b, dy)
    leaves = [v.requires_grad_() for v in (x, w, b)]
    y = autograd.layer_norm(*leaves)
    got = torch.autograd.grad(y, leaves, dy.requires_grad_(), create_graph=True)        # (torch refuses where the incoming gradient has one)
    check([y, *got], want, tol)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        got[0].sum().backward()


@gpu
def test_statistics_of_two_calls_and_saved_rows(device):
    """Two passes in flight keep statistics of their own, in whichever order their gradients are taken, and no rows at all give zero gradients."""
    from craft_amd import autograd
    runs = []
    for seed in (0, 1):
        x, w, b, dy = make("fp16", 30 + seed, 130, seed)
        want = norm64(x, w, b, dy)
        leaves = [v.requires_grad_() for v in (x, w, b)]
        runs.append((leaves, dy, want, autograd.layer_norm(*leaves)))
    for leaves, dy, (want, tol), y in runs[::-1]:
        check([y, *torch.autograd.grad(y, leaves, dy)], want, tol)
    x, w = torch.zeros(0, 130, device="cuda", requires_grad=True), torch.ones(130, device="cuda", requires_grad=True)
    gx, gw = torch.autograd.grad(autograd.layer_norm(x, w), (x, w), torch.zeros(0, 130, device="cuda"))
    assert gx.shape == (0, 130) and not gw.any()


@gpu
def test_out_that_shares_memory(device):
    """x itself and columns beside it are written; rows that others still read are refused."""
    from craft_amd import ops
    from craft_amd.hip import CraftHipError
    buf = torch.randn(50, 300, device="cuda")
    want = ops.layer_norm(buf[:, :130])
    assert torch.equal(ops.layer_norm(buf[:, :130], out=buf[:, 130:260]), want)
    for x, out in ((buf[:40, :100], buf[1:41, :100]), (buf[:, :100], buf[:, 50:150]), (buf[:1, :100].expand(40, 100), buf[:40, :100])):
        with pytest.raises(CraftHipError, match="must not overlap"):
            ops.layer_norm(x, out=out)
    assert torch.equal(ops.layer_norm(buf[:, :130], out=buf[:, :130]), want)
    one = buf[:1, 200:].clone()
    assert torch.equal(ops.layer_norm(one, out=one), ops.layer_norm(buf[:1, 200:]))
