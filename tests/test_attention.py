"""ops.attention / autograd.attention against the formula in 64 bits: types, head layouts, lengths, masks, strides, and what they refuse."""
import math

import pytest
import torch

from attention_reference import attention64, check, visible

gpu = pytest.mark.gpu
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def make(t, B, nq, nk, H, Hk, D, seed=0, spread=3.0, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)                            # noqa: E731
    return [x.to(TYPES[t]).to(device) for x in (spread * n(B, nq, H, D), n(B, nk, Hk, D), n(B, nk, Hk, D), n(B, nq, H, D))]


def slopes_of(H, device="cuda"):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device=device)


def doc_ids(B, n, pieces, padding, seed=0, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    out = torch.full((B, n), -1, dtype=torch.int32)
    for b in range(B):
        m = n - padding
        cut = sorted({0, m, *torch.randint(0, m + 1, (pieces - 1,), generator=g).tolist()})
        for d, (a, e) in enumerate(zip(cut, cut[1:])):
            out[b, a:e] = d
    return out.to(device)


def both(t, B, nq, nk, H, Hk, D, seed=0, spread=3.0, **how):
    """The differentiable form with its gradients and the inference form, each against 64 bits."""
    from craft_amd import autograd, ops
    q, k, v, go = make(t, B, nq, nk, H, Hk, D, seed, spread)
    res, tol = attention64(q, k, v, go, **how)
    q, k, v = (x.requires_grad_() for x in (q, k, v))
    o = autograd.attention(q, k, v, **how)
    check([o, *torch.autograd.grad(o, (q, k, v), go)], res, tol)
    check([ops.attention(q, k, v, **how)], res[:1], tol[:1])


# ---------------------------------------------------------------------------------------------------------------- CPU: the oracle and the refusals
def test_reference_gradients_are_autograds():
    """The formulas the kernels are held to, against torch's own differentiation of the definition."""
    q, k, v, go = make("fp32", 2, 9, 13, 4, 2, 8, device="cpu")
    how = dict(cap=4.0, slopes=slopes_of(4, "cpu"), causal=True, prefix=torch.tensor([0, 7], dtype=torch.int32))
    res, _ = attention64(q, k, v, go, **how)
    a, b, c = (x.double().requires_grad_() for x in (q, k, v))
    kk, vv = (x.transpose(1, 2).repeat_interleave(2, 1) for x in (b, c))
    z = 4.0 * torch.tanh(a.transpose(1, 2) @ kk.mT / math.sqrt(8) / 4.0)
    z = z - slopes_of(4, "cpu").double()[:, None, None] * ((torch.arange(9)[:, None] + 4) - torch.arange(13)).abs()
    o = (torch.softmax(z.masked_fill(~visible(9, 13, True, how["prefix"], batch=2)[:, None], -math.inf), -1) @ vv).transpose(1, 2)
    for r, g in zip(res, (o, *torch.autograd.grad(o, (a, b, c), go.double()))):
        assert torch.allclose(r, g, rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("change, says", [
    (dict(q=torch.zeros(1, 4, 3, 16), k=torch.zeros(1, 4, 2, 16), v=torch.zeros(1, 4, 2, 16)), "no multiple"),
    (dict(q=torch.zeros(1, 4, 2, 12), k=torch.zeros(1, 4, 2, 12), v=torch.zeros(1, 4, 2, 12)), "multiple of 8"),
    (dict(q=torch.zeros(1, 4, 2, 136), k=torch.zeros(1, 4, 2, 136), v=torch.zeros(1, 4, 2, 136)), "multiple of 8"),
    (dict(k=torch.zeros(1, 4, 2, 8)), "do not fit"),
    (dict(v=torch.zeros(1, 5, 2, 16)), "do not fit"),
    (dict(q=torch.zeros(4, 2, 16)), "are \\[batch"),
    (dict(k=torch.zeros(1, 4, 2, 16, dtype=torch.float16)), "one type"),
    (dict(q=torch.zeros(1, 4, 2, 16).double(), k=torch.zeros(1, 4, 2, 16).double(), v=torch.zeros(1, 4, 2, 16).double()), "one type"),
    (dict(cap=-1.0), "cap"), (dict(cap=float("nan")), "cap"), (dict(cap=float("inf")), "cap"),
    (dict(cap=1e-38), "scale / cap"), (dict(cap=1e-20, scale=1e15), "scale / cap"),
    (dict(q=torch.zeros(1, 4, 2, 16).half(), k=torch.zeros(1, 4, 2, 16).half(), v=torch.zeros(1, 4, 2, 16).half(), cap=4097.0), "4096"),
    (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(prefix=torch.zeros(1, dtype=torch.int32)), "causal=True"),
    (dict(prefix=torch.zeros(2, dtype=torch.int32), causal=True), "prefix must"),
    (dict(prefix=torch.zeros(1, dtype=torch.int64), causal=True), "prefix must"),
    (dict(slopes=torch.zeros(3)), "slopes"), (dict(slopes=torch.zeros(2).half()), "slopes"),
    (dict(slopes=torch.zeros(2, requires_grad=True)), "no gradient"),
    (dict(docs=torch.zeros(1, 3, dtype=torch.int32)), "docs must"),
    (dict(docs=torch.zeros(1, 4)), "docs must"),
    (dict(docs_k=torch.zeros(1, 4, dtype=torch.int32)), "needs docs"),
    (dict(docs=torch.zeros(1, 4, dtype=torch.int32), docs_k=torch.zeros(1, 3, dtype=torch.int32)), "docs_k must"),
    (dict(q=torch.zeros(1, 3, 2, 16), docs=torch.zeros(1, 3, dtype=torch.int32)), "docs_k too"),
    (dict(), "device tensors"),
])
def test_refusals(change, says):
    from craft_amd import autograd, ops
    from craft_amd.hip import CraftHipError
    args = dict(q=torch.zeros(1, 4, 2, 16), k=torch.zeros(1, 4, 2, 16), v=torch.zeros(1, 4, 2, 16), **{})
    args.update(change)
    q, k, v = args.pop("q"), args.pop("k"), args.pop("v")
    with torch.enable_grad(), pytest.raises(CraftHipError, match=says):
        autograd.attention(q, k, v, **args)
    if says != "no gradient":                                             # (without gradients, slopes that have one are a plain input)
        with pytest.raises(CraftHipError, match=says):
            ops.attention(q, k, v, **args)


def test_entry_points_check_their_arguments():
    """The C entry points refuse what their kernels assume, before anything is launched (no GPU needed)."""
    import ctypes

    from craft_amd import hip
    lib = hip.load()
    buf = 4096                                                             # an aligned address that is never read: every call below is refused first
    good = [1, 4, 4, 2, 2, 16] + [128, 32, 16] * 4

    def fwd(shape=good, q=buf, k=buf, v=buf, out=buf, scale=1.0, cap=0.0, causal=0, dtype=2, splits=0, docs=(None, None), prefix=None, ws=None, ws_bytes=0, lse=None, rest=None):
        return lib.craft_attention_fwd(q, k, v, (ctypes.c_long * len(shape))(*shape), None, prefix, docs[0], docs[1], scale, cap, causal, dtype, splits, out, lse,
                                       rest, ws, ws_bytes, None)

    def with_(i, x):
        s = list(good)
        s[i] = x
        return s
    ARG, ALIGN, UNSUPPORTED = 10001, 10002, 10003
    assert fwd(with_(0, 0)) == UNSUPPORTED and fwd(with_(1, -1)) == UNSUPPORTED and fwd(with_(2, 1 << 29)) == UNSUPPORTED
    assert fwd(with_(3, 3)) == UNSUPPORTED and fwd(with_(5, 136)) == UNSUPPORTED and fwd(with_(5, 20)) == ALIGN
    assert fwd(with_(7, 36)) == ALIGN and fwd(with_(10, -16)) == ALIGN and fwd(with_(10, 1 << 23)) == UNSUPPORTED
    assert fwd(q=buf + 8) == ALIGN and fwd(k=None) == ALIGN and fwd(out=buf + 2) == ALIGN
    assert fwd(dtype=3) == ARG and fwd(cap=-1.0) == ARG and fwd(cap=float("nan")) == ARG and fwd(scale=float("nan")) == ARG
    assert fwd(dtype=2, cap=4097.0) == UNSUPPORTED and fwd(dtype=2, cap=1e-38) == ARG and fwd(with_(1, 1 << 21), splits=1) == UNSUPPORTED
    assert fwd(docs=(buf, None)) == ARG and fwd(docs=(buf, buf)) == ARG                      # (no workspace for the ranges)
    assert fwd(prefix=buf) == ARG and fwd(splits=-1) == ARG and fwd(splits=2) == ARG and fwd(splits=1, lse=buf) == ARG and fwd(splits=1, rest=buf) == ARG and fwd(rest=buf + 8) == ARG
    shape5 = (ctypes.c_long * 21)(*(good + [128, 32, 16]))
    bwd = lambda ws, n, lse=buf, dk=buf: lib.craft_attention_bwd(buf, buf, buf, buf, None, lse, buf, shape5, None, None, None, None, 1.0, 0.0, 0, 2, 1, buf, dk, buf, ws, n, None)  # noqa: E731
    assert bwd(None, 0) == ARG and bwd(buf, 31) == ARG and bwd(buf, 1 << 20, lse=None) == ARG and bwd(buf, 1 << 20, dk=buf + 4) == ALIGN


# ---------------------------------------------------------------------------------------------------------------- GPU
SHAPES = [  # B, queries, keys, heads, key heads, width
    (1, 1, 1, 1, 1, 8), (2, 2, 2, 2, 1, 16), (1, 31, 33, 2, 2, 32), (1, 64, 64, 1, 1, 40), (2, 65, 65, 3, 3, 64), (1, 127, 129, 2, 1, 72),
    (1, 130, 130, 4, 2, 128), (2, 1, 300, 8, 2, 128), (1, 5, 77, 4, 4, 64), (1, 200, 40, 2, 2, 64), (1, 300, 300, 6, 2, 24), (1, 40, 530, 12, 1, 64)]


@gpu
@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_plain(device, t, shape):
    both(t, *shape)


@gpu
@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_causal_capped_biased(device, t, shape):
    """All at once; more queries than keys leaves the first rows empty."""
    both(t, *shape, causal=True, cap=5.0, slopes=slopes_of(shape[3]))


@gpu
@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("cap, slopes, causal", [(0.0, True, False), (30.0, False, False), (2.0, True, False), (0.0, True, True), (0.0, False, True)])
def test_one_by_one(device, t, cap, slopes, causal):
    both(t, 2, 150, 150, 4, 2, 64, cap=cap, slopes=slopes_of(4) if slopes else None, causal=causal)


@gpu
@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("nq, nk, prefix", [(150, 150, [0, 150]), (70, 200, [1, 131]), (33, 33, [500, 17]), (140, 20, [3, 0]), (1, 90, [90, 4]), (140, 140, [64, 63])])
def test_prefix(device, t, nq, nk, prefix):
    both(t, 2, nq, nk, 4, 2, 64, causal=True, prefix=torch.tensor(prefix, dtype=torch.int32, device="cuda"))


@gpu
@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("n, pieces, padding", [(33, 1, 0), (65, 3, 7), (200, 5, 0), (300, 9, 140), (300, 2, 299), (128, 128, 0), (40, 1, 40)])
@pytest.mark.parametrize("causal", [False, True])
def test_documents(device, t, n, pieces, padding, causal):
    both(t, 2, n, n, 4, 2, 64, causal=causal, docs=doc_ids(2, n, pieces, padding))


@gpu
@pytest.mark.parametrize("t", list(TYPES))
def test_documents_out_of_order(device, t):
    """Interleaved documents (no sorted runs), other ids for queries and keys, queries whose document no key has."""
    g = torch.Generator().manual_seed(5)
    dq = torch.randint(-1, 6, (2, 90), generator=g, dtype=torch.int32).cuda()
    dk = torch.randint(-1, 5, (2, 210), generator=g, dtype=torch.int32).cuda()
    both(t, 2, 90, 210, 4, 2, 64, docs=dq, docs_k=dk)
    both(t, 2, 90, 210, 4, 2, 64, docs=dq, docs_k=dk, causal=True, prefix=torch.tensor([40, 0], dtype=torch.int32, device="cuda"), cap=3.0)
    both(t, 2, 3, 210, 4, 2, 64, docs=dq[:, :3].contiguous(), docs_k=dk)


@gpu
@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("nq", [1, 100])
def test_padding_may_hold_anything(device, t, nq):
    """inf and NaN in rows whose document is negative reach nothing, in the results and in the gradients; the padded rows' own are zero."""
    from craft_amd import autograd, ops
    q, k, v, go = make(t, 2, nq, 100, 4, 2, 64)
    dk = doc_ids(2, 100, 3, 30)
    dq = dk[:, -nq:].contiguous() if nq > 1 else torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    res, tol = attention64(q, k, v, go, docs=dq, docs_k=dk)
    bad = torch.tensor([math.nan, math.inf, -math.inf], device="cuda").to(q.dtype)
    for x, d in ((q, dq), (go, dq), (k, dk), (v, dk)):
        m = (d < 0)[:, :, None, None].expand(x.shape)
        x[m] = bad[torch.arange(int(m.sum()), device="cuda") % 3]
    q, k, v = (x.requires_grad_() for x in (q, k, v))
    o = autograd.attention(q, k, v, docs=dq, docs_k=dk)
    grads = torch.autograd.grad(o, (q, k, v), go)
    check([o, *grads], res, tol)
    check([ops.attention(q, k, v, docs=dq, docs_k=dk)], res[:1], tol[:1])
    assert not grads[0][dq < 0].any() and not grads[1][dk < 0].any() and not grads[2][dk < 0].any() and not o[dq < 0].any()


@gpu
@pytest.mark.parametrize("t", list(TYPES))
def test_large_scores(device, t):
    """Scores in the hundreds: the running maximum carries the sums; a cap brings them back."""
    both(t, 1, 140, 140, 2, 2, 64, spread=60.0)
    both(t, 1, 140, 140, 2, 2, 64, spread=60.0, cap=20.0, causal=True)
    both(t, 1, 140, 140, 2, 2, 64, scale=-0.3)


@gpu
def test_rising_scores(device):
    """Every later key tile raises the maximum: the output is rescaled each time."""
    from craft_amd import ops
    q = torch.ones(1, 4, 1, 32, device="cuda", dtype=torch.bfloat16)
    k = (torch.arange(512, device="cuda").float()[None, :, None, None] / 8).expand(1, 512, 1, 32).to(torch.bfloat16)
    v = torch.randn(1, 512, 1, 32, device="cuda").bfloat16()
    for n in (4, 100):
        qq = q[:, :1].expand(1, n, 1, 32).contiguous()
        res, tol = attention64(qq, k, v, scale=1.0)
        check([ops.attention(qq, k, v, scale=1.0)], res, tol)


@gpu
def test_views(device):
    """Slices of one packed projection, a head-major layout, expanded heads, and rows that no 16-byte step fits are read right."""
    from craft_amd import autograd, ops
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn(2, 70, 3, 4, 64, generator=g).half().cuda()
    q, k, v = qkv.unbind(2)
    res, tol = attention64(q, k, v, causal=True)
    check([ops.attention(q, k, v, causal=True)], res, tol)
    hm = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
    check([ops.attention(*hm, causal=True)], res, tol)
    odd = torch.randn(2 * 70 * 4 * 67 + 5, generator=g).half().cuda()
    odd = [torch.as_strided(odd, (2, 70, 4, 64), (70 * 4 * 67, 4 * 67, 67, 1), i) for i in (1, 3, 5)]
    res, tol = attention64(*odd)
    check([ops.attention(*odd)], res, tol)
    k1, v1 = (x[:, :, :1].expand(2, 70, 4, 64) for x in (k, v))
    res, tol = attention64(q, k1, v1)
    check([ops.attention(q, k1, v1)], res, tol)
    out = torch.zeros(2, 70, 8, 64, device="cuda", dtype=torch.float16)
    assert ops.attention(q, k1, v1, out=out[:, :, 2:6]).data_ptr() == out[:, :, 2:6].data_ptr()
    check([out[:, :, 2:6]], res, tol)
    assert not out[:, :, :2].any() and not out[:, :, 6:].any()
    # gradients through views, and a gradient that is an expanded scalar
    leaf = qkv.clone().requires_grad_()
    autograd.attention(*leaf.unbind(2), causal=True).sum().backward()
    res, tol = attention64(q, k, v, torch.ones_like(q), causal=True)
    check([res[0], *leaf.grad.unbind(2)], res, tol)


@gpu
def test_lengths_of_zero(device):
    from craft_amd import autograd, ops
    for nq, nk, B in ((0, 5, 1), (5, 0, 1), (5, 5, 0)):
        q, k, v, go = make("bf16", B, nq, nk, 4, 2, 64)
        assert ops.attention(q, k, v).shape == q.shape and not ops.attention(q, k, v).any()
        q, k, v = (x.requires_grad_() for x in (q, k, v))
        for g, x in zip(torch.autograd.grad(autograd.attention(q, k, v), (q, k, v), go), (q, k, v)):
            assert g.shape == x.shape and not g.any()


@gpu
def test_long_cache_past_32_bits(device):
    """Keys and values that lie more than 2^32 bytes behind the first: only the last one scores above the others."""
    from craft_amd import ops
    nk, Hk, D = (1 << 20) + 77, 18, 128                                    # 4.8 GB each
    k = torch.zeros(1, nk, Hk, D, device="cuda", dtype=torch.bfloat16)
    v = torch.zeros(1, nk, Hk, D, device="cuda", dtype=torch.bfloat16)
    last = torch.randn(Hk, D, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    k[0, -1], v[0, -1] = 8.0, last
    q = torch.full((1, 1, Hk, D), 8.0, device="cuda", dtype=torch.bfloat16)
    o = ops.attention(q, k, v, causal=True)
    assert torch.equal(o[0, 0], last)                                      # exp(-724) of the rest
    o = ops.attention(q.expand(1, 130, Hk, D), k, v, causal=True)          # the block kernel: only the last query sees the last key
    assert torch.equal(o[0, -1], last) and not o[0, :-1].any()


@gpu
def test_gradients_against_differences(device):
    """The fp32 gradients against central differences of the kernel's own forward pass, along random directions.  An fp32 sum of 2 880 products of
    unit size is off by at most 1e-4; over a step of 2e-2 that is 1e-2 of a derivative of size 10 to 100, and the cubic term is below it."""
    from craft_amd import autograd
    q, k, v, go = make("fp32", 1, 45, 45, 2, 1, 32, spread=1.0)
    how = dict(cap=3.0, causal=True, slopes=slopes_of(2))
    q, k, v = (x.requires_grad_() for x in (q, k, v))
    grads = torch.autograd.grad(autograd.attention(q, k, v, **how), (q, k, v), go)
    for n, x in enumerate((q, k, v)):
        d = torch.randn(x.shape, generator=torch.Generator().manual_seed(n)).cuda()
        f = lambda s: (autograd.attention(*[y.detach() + (s * d if m == n else 0) for m, y in enumerate((q, k, v))], **how).double() * go.double()).sum().item()  # noqa: E731,B023
        num = (f(1e-2) - f(-1e-2)) / 2e-2
        assert abs(num - (grads[n].double() * d.double()).sum().item()) < 2e-2 * max(1.0, abs(num))


@gpu
@pytest.mark.parametrize("t", ["bf16", "fp32"])
def test_same_bits_every_time(device, t):
    """No result depends on the order of blocks or atomics: shared heads, split keys and all."""
    from craft_amd import autograd, ops
    q, k, v, go = make(t, 2, 260, 260, 8, 2, 64)
    q, k, v = (x.requires_grad_() for x in (q, k, v))
    runs = []
    for _ in range(3):
        o = autograd.attention(q, k, v, causal=True)
        runs.append([o, *torch.autograd.grad(o, (q, k, v), go), ops.attention(q[:, :1], k, v)])
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(runs[0], r))


@gpu
def test_other_stream_and_captured(device):
    """On a side stream, and captured into a graph whose replays follow new inputs (single tokens, whole rows, with documents), each against eager."""
    from craft_amd import ops
    q, k, v, _ = make("fp16", 2, 130, 130, 4, 2, 64)
    docs = doc_ids(2, 130, 4, 10)
    want = ops.attention(q, k, v, docs=docs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.attention(q, k, v, docs=docs)
    side.synchronize()
    assert torch.equal(got, want)
    one = q[:, -1:].contiguous()
    with torch.cuda.stream(side):                                          # (warm-up outside the capture)
        ops.attention(q, k, v, docs=docs), ops.attention(one, k, v, causal=True)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a = ops.attention(q, k, v, docs=docs)
        b = ops.attention(one, k, v, causal=True)
    for seed in range(4):
        for x, y in zip((q, k, v), make("fp16", 2, 130, 130, 4, 2, 64, seed=seed)):
            x.copy_(y)
        docs.copy_(doc_ids(2, 130, 4, 10, seed=seed))
        one.copy_(q[:, -1:])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, ops.attention(q, k, v, docs=docs)) and torch.equal(b, ops.attention(one, k, v, causal=True))


@gpu
@pytest.mark.parametrize("t, cap", [("fp16", 4096.0), ("bf16", 4096.0), ("fp32", 1e6), ("fp32", 1e-3), ("bf16", 1e-3)])
def test_largest_and_smallest_caps(device, t, cap):
    """A cap far above every score changes none of them (16-bit types: by cap 2^-22 = 2^-10 of a power of two at most, an eighth of a bf16 rounding and
    half of an fp16 one of each probability); one far below leaves their signs."""
    from craft_amd import ops
    q, k, v, _ = make(t, 1, 70, 70, 2, 2, 32)
    a, b = ops.attention(q, k, v, cap=cap).double().cpu(), attention64(q, k, v, cap=cap)[0][0]
    eps = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8, "fp32": 2.0 ** -21}[t]
    # the probabilities are off by their rounding and twice the scores' error (their own and the sum's), the result by that of sum p |v|, and rounded once
    size = attention64(q, k, v.abs(), cap=cap)[0][0]
    score = 2.0 ** -10 if t != "fp32" else 2.0 ** -19          # fp32: products of 32 terms of unit size times 3, and two roundings of scores up to 30
    assert ((a - b).abs() <= (2 * eps + 2 * score) * size + 2.0 ** -25).all()


@gpu
def test_out_in_place_of_q_and_refused(device):
    from craft_amd import ops
    from craft_amd.hip import CraftHipError
    for nq in (150, 1):                                        # (blocks of queries, and single tokens whose keys are split)
        q, k, v, _ = make("bf16", 2, nq, 700, 4, 2, 64)
        want = ops.attention(q, k, v, causal=True)
        assert ops.attention(q, k, v, causal=True, out=q) is q and torch.equal(q, want)
    q, k, v, _ = make("bf16", 1, 40, 40, 2, 2, 64)
    for out in (k, v, torch.empty(1, 40, 1, 64, device="cuda", dtype=q.dtype).expand(1, 40, 2, 64)):
        with pytest.raises(CraftHipError, match="out must"):
            ops.attention(q, k, v, out=out)


@gpu
def test_without_gradients_is_the_serving_form(device):
    """autograd.attention and layer_norm under no_grad give the bits of ops'."""
    from craft_amd import autograd, ops
    q, k, v, _ = make("bf16", 2, 1, 500, 4, 2, 64)
    with torch.no_grad():
        assert torch.equal(autograd.attention(q, k, v, causal=True), ops.attention(q, k, v, causal=True))
        x = torch.randn(5, 70, device="cuda")
        assert torch.equal(autograd.layer_norm(x), ops.layer_norm(x))


@gpu
def test_two_streams_at_once(device):
    """Calls that run beside each other share nothing: each has its own workspace."""
    from craft_amd import autograd
    a, b = (make("bf16", 1, 300, 300, 4, 2, 64, seed=s) for s in (1, 2))
    docs = doc_ids(1, 300, 3, 9)

    def run(x):
        leaves = [y.clone().requires_grad_() for y in x[:3]]
        o = autograd.attention(*leaves, causal=True, cap=20.0, docs=docs)
        return [o, *torch.autograd.grad(o, leaves, x[3])]
    want = [run(a), run(b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(4):
        got = []
        for s, x in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                got.append(run(x))
        torch.cuda.synchronize()
        for w, g in zip(want, got):
            assert all(torch.equal(m, n) for m, n in zip(w, g))


def offset(x, by=1):
    """x's values, contiguous, at an address that no 16-byte load fits."""
    flat = torch.empty(x.numel() + by, device=x.device, dtype=x.dtype)
    t = flat[by:].view(x.shape)
    t.copy_(x)
    return t


@pytest.mark.parametrize("t", list(TYPES))
def test_contiguous_but_misaligned_is_copied(t):
    """A slice of a flat buffer is contiguous wherever it starts: contiguous() hands it back as it is."""
    from craft_amd import ops
    x = make(t, 2, 5, 5, 2, 2, 16, device="cpu")[0]
    y = offset(x)
    assert y.is_contiguous() and y.data_ptr() % 16
    z = ops._strided(y)
    assert z.data_ptr() % 16 == 0 and torch.equal(z, x)
    a = offset(x, 16)                                                      # (32 or 64 bytes on: nothing to copy)
    assert ops._strided(a) is a


@gpu
@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("nq", [1, 50])
def test_misaligned_inputs_and_gradients(device, t, nq):
    from craft_amd import autograd, ops
    from craft_amd.hip import CraftHipError
    q, k, v, go = make(t, 2, nq, 50, 4, 2, 40)
    res, tol = attention64(q, k, v, go, causal=True)
    q, k, v = (offset(x).requires_grad_() for x in (q, k, v))
    o = autograd.attention(q, k, v, causal=True)
    check([o, *torch.autograd.grad(o, (q, k, v), offset(go))], res, tol)
    check([ops.attention(q, k, v, causal=True)], res[:1], tol[:1])
    with pytest.raises(CraftHipError, match="out must"):
        ops.attention(q, k, v, out=offset(go))


WIDTHS = [32, 72, 128]                                                     # (64 is every other test's; 72 and 128: V in LDS, 32-row tiles, columns behind D)


@gpu
@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("D", WIDTHS)
@pytest.mark.parametrize("causal", [False, True])
def test_documents_at_every_width(device, t, D, causal):
    """Whole 128-key blocks of padding, which no query tile meets, among them."""
    both(t, 2, 650, 650, 4, 2, D, causal=causal, docs=doc_ids(2, 650, 5, 270), cap=8.0 if causal else 0.0, slopes=None if causal else slopes_of(4))
    both(t, 1, 300, 300, 2, 2, D, causal=causal, docs=doc_ids(1, 300, 60, 1))


@gpu
@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("D", WIDTHS)
def test_prefix_at_every_width(device, t, D):
    for nq, nk, prefix in ((300, 300, [130, 0]), (140, 20, [3, 0]), (70, 400, [1, 395])):
        both(t, 2, nq, nk, 4, 2, D, causal=True, prefix=torch.tensor(prefix, dtype=torch.int32, device="cuda"))


@gpu
@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("D", WIDTHS)
def test_padding_may_hold_anything_at_every_width(device, t, D):
    """As test_padding_may_hold_anything, with padding in front, in the middle and over whole tiles and blocks, queries and keys apart."""
    from craft_amd import autograd, ops
    nq, nk = 330, 410
    q, k, v, go = make(t, 2, nq, nk, 4, 2, D)
    dq, dk = doc_ids(2, nq, 3, 140), doc_ids(2, nk, 3, 150)
    dq[1], dk[1] = dq[1].roll(37), dk[1].roll(70)
    dq[0, 50:53], dk[0, 20:90] = -7, -2147483648
    res, tol = attention64(q, k, v, go, docs=dq, docs_k=dk, causal=True)
    bad = torch.tensor([math.nan, math.inf, -math.inf], device="cuda").to(q.dtype)
    for x, d in ((q, dq), (go, dq), (k, dk), (v, dk)):
        m = (d < 0)[:, :, None, None].expand(x.shape)
        x[m] = bad[torch.arange(int(m.sum()), device="cuda") % 3]
    q, k, v = (x.requires_grad_() for x in (q, k, v))
    o = autograd.attention(q, k, v, docs=dq, docs_k=dk, causal=True)
    grads = torch.autograd.grad(o, (q, k, v), go)
    check([o, *grads], res, tol)
    check([ops.attention(q, k, v, docs=dq, docs_k=dk, causal=True)], res[:1], tol[:1])
    assert not grads[0][dq < 0].any() and not grads[1][dk < 0].any() and not grads[2][dk < 0].any() and not o[dq < 0].any()


@gpu
@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("B, nq, nk, H, Hk, D, how", [
    (64, 100, 100, 16, 8, 64, {}), (43, 150, 260, 12, 4, 128, dict(causal=True, cap=6.0, slopes=True)), (43, 150, 260, 12, 4, 40, dict(docs=True)),
    (43, 70, 260, 8, 4, 128, dict(docs=True, causal=True, slopes=True)), (86, 40, 330, 6, 2, 24, dict(causal=True, prefix=True, slopes=True))])
def test_one_block_for_a_group_of_heads(device, t, B, nq, nk, H, Hk, D, how):
    """Batches that fill the card with one block for each key head: it walks over the query heads of its group, each with its slope and log-sums."""
    from craft_amd import autograd
    assert B * Hk * ((nk + 127) // 128) >= 512 and H > Hk
    how = dict(how)
    if how.get("slopes"):
        how["slopes"] = slopes_of(H)
    if how.get("prefix"):
        how["prefix"] = torch.arange(B, dtype=torch.int32, device="cuda") * 4
    if how.pop("docs", False):
        d = doc_ids(B, nk, 5, 130)
        how.update(docs=d[:, :nq].contiguous(), docs_k=d)
    q, k, v, go = make(t, B, nq, nk, H, Hk, D)
    res, tol = attention64(q, k, v, go, **how)
    q, k, v = (x.requires_grad_() for x in (q, k, v))
    o = autograd.attention(q, k, v, **how)
    check([o, *torch.autograd.grad(o, (q, k, v), go)], res, tol)


def unavoidable(exact, t):
    """What rounding the exact result to the type costs, in the mean."""
    return (exact.to(t).double() - exact).norm().item()


@gpu
@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("D, size", [(64, 1.0), (64, 1e-3), (64, 1e-5), (128, 1e-4), (72, 1e-5), (32, 3000.0), (128, 3000.0)])
def test_gradients_of_every_size(device, t, D, size):
    """Gradients keep their bits whatever the size of the loss', in 16 bits too.  The bounds are those of gradients of unit size times the size (a power of two
    near it), and half of fp16's smallest step for the last rounding; and in the mean: a rounding is off by its half step u / sqrt 3 at the worst, by 0.43 u over
    all mantissas, so operands rounded once (incoherent, every term by itself) and a result rounded once are off by sqrt(1 + (0.577 / 0.43)^2) = 1.7 times what
    rounding the result alone costs (fp32: the elements' bounds alone; its operands are not rounded)."""
    from craft_amd import autograd
    q, k, v, go = make(t, 1, 700, 700, 4, 2, D)
    s = 2.0 ** round(math.log2(size))
    how = dict(causal=True, slopes=slopes_of(4)) if D == 64 else dict(cap=20.0) if D == 128 else {}
    go = (go.double() * s).to(go.dtype)                                    # (1e-5 in fp16: below its smallest normal number, rounded once more)
    res, tol = attention64(q, k, v, go.double() / s, **how)
    res, tol = [res[0]] + [r * s for r in res[1:]], [tol[0]] + [e * s + 2.0 ** -25 * (t == "fp16") for e in tol[1:]]
    assert max(r.abs().max() for r in res) < 6e4
    q, k, v = (x.requires_grad_() for x in (q, k, v))
    o = autograd.attention(q, k, v, **how)
    got = [o, *torch.autograd.grad(o, (q, k, v), go)]
    check(got, res, tol)
    for g, r, name in zip(got[1:], res[1:], ("dq", "dk", "dv")):
        off, least = (g.cpu().double() - r).norm().item(), unavoidable(r, TYPES[t])
        assert t == "fp32" or off <= 2.0 * least, (name, off / least)


def two_keys_each(D, n=200, device="cuda"):
    """Every query looks at two keys whose values differ widely: gradients of scores past fp16's largest number, of everything else within it."""
    _, k, v, go = make("fp16", 1, n, n, 1, 1, D, device=device)
    scale = 6.0 / (4 * D)
    q = (4 * (k.float() + k.float().roll(1, 1))).half()
    return q, k, (v.float() * 24 * (64 / D) ** 0.5).half(), (go.float() * 1000).half(), scale


@pytest.mark.parametrize("D", [64, 128])
def test_two_keys_each(D):
    q, k, v, go, scale = two_keys_each(D, device="cpu")
    res, _ = attention64(q, k, v, go, scale=scale)
    p = torch.softmax(scale * q.double()[0, :, 0] @ k.double()[0, :, 0].T, -1)
    dp = go.double()[0, :, 0] @ v.double()[0, :, 0].T
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    assert ds.abs().max() > 2 * 65504 and max(r.abs().max() for r in res) < 6e4


@gpu
@pytest.mark.parametrize("D", [64, 128])
def test_score_gradients_past_the_largest_fp16(device, D):
    from craft_amd import autograd
    q, k, v, go, scale = two_keys_each(D)
    res, tol = attention64(q, k, v, go, scale=scale)
    q, k, v = (x.requires_grad_() for x in (q, k, v))
    o = autograd.attention(q, k, v, scale=scale)
    check([o, *torch.autograd.grad(o, (q, k, v), go)], res, tol)


@gpu
@pytest.mark.parametrize("D", [64, 128])
def test_small_probabilities_keep_their_bits(device, D):
    """Flat rows of 20000 keys: probabilities of 5e-5, below fp16's smallest normal number, and score gradients of 1e-8."""
    from craft_amd import autograd
    q, k, v, go = make("fp16", 1, 130, 20000, 1, 1, D, spread=0.05)
    go = go * 1e-3
    s = 2.0 ** -10
    res, tol = attention64(q, k, v, go.double() / s)
    res, tol = [res[0]] + [r * s for r in res[1:]], [tol[0]] + [e * s + 2.0 ** -25 for e in tol[1:]]
    q, k, v = (x.requires_grad_() for x in (q, k, v))
    o = autograd.attention(q, k, v)
    got = [o, *torch.autograd.grad(o, (q, k, v), go)]
    check(got, res, tol)
    for g, r, name in zip(got[1:], res[1:], ("dq", "dk", "dv")):
        off, least = (g.cpu().double() - r).norm().item(), unavoidable(r, torch.float16)
        assert off <= 2.0 * least, (name, off / least)


@gpu
@pytest.mark.parametrize("t", list(TYPES))
def test_infinite_gradients_show(device, t):
    """An overflow of the loss reaches every gradient that depends on it, where a loss scale looks for it.  (Finite values are what the operator asks for:
    nothing says where else it goes.)"""
    from craft_amd import autograd
    q, k, v, go = make(t, 1, 300, 300, 4, 2, 64)
    for bad in (math.inf, math.nan):
        go[0, 130, 1, 3] = bad
        a = [x.clone().requires_grad_() for x in (q, k, v)]
        dq, dk, dv = torch.autograd.grad(autograd.attention(*a), a, go)
        assert not torch.isfinite(dq[0, 130, 1]).any() and not torch.isfinite(dk[0, :, 0]).any() and not torch.isfinite(dv[0, :, 0, 3]).any()
        assert torch.isfinite(dq[0, :130]).all()


def test_gradients_workspace_is_checked():
    """fp16 asks for the room of its powers of two; the other types do not."""
    import ctypes

    from craft_amd import hip
    lib, buf = hip.load(), 4096
    shape = (ctypes.c_long * 21)(*([2, 5, 4, 6, 3, 16] + [128, 32, 16] * 5))
    bwd = lambda dtype, n, group=0: lib.craft_attention_bwd(buf, buf, buf, buf, None, buf, buf, shape, None, None, None, None, 1.0, 0.0, 0, dtype, group, buf, buf, buf, buf, n, None)  # noqa: E731
    row, part = 240, 2 * 2 * 4 * 6 * 16 * 4
    assert bwd(2, row + 48 - 1) == 10001 and bwd(2, row + 48 + part - 1, 1) == 10001          # (10 rows of a key head: one slice, of 6 key heads)
    assert bwd(1, row - 1) == 10001 and bwd(0, row + part - 1, 1) == 10001


def calls_of(monkeypatch):
    """The names and arguments of the package's calls into the library from here on."""
    from craft_amd import ops
    seen, call = [], ops.call
    monkeypatch.setattr(ops, "call", lambda name, *a: (seen.append((name, a)), call(name, *a))[1])
    return seen


@pytest.mark.parametrize("training", [False, True])
def test_inputs_without_gradients_take_the_serving_form(monkeypatch, training):
    """Gradients enabled and nothing that needs one: what a server that forgets no_grad calls."""
    from craft_amd import autograd, ops
    took = []
    for name in ("attention", "layer_norm"):
        monkeypatch.setattr(ops, name, lambda *a, n=name, **k: took.append(n))
    for cls in (autograd.Attention, autograd.LayerNorm):
        monkeypatch.setattr(cls, "apply", lambda *a, n=cls.__name__: took.append(n))
    x, w = torch.zeros(1, 4, 2, 16), torch.zeros(16, requires_grad=training)
    with torch.enable_grad():
        autograd.attention(x, x, x.clone().requires_grad_(training))
        autograd.layer_norm(x, None, w)
    assert took == (["Attention", "LayerNorm"] if training else ["attention", "layer_norm"])


@gpu
@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("H, Hk", [(4, 4), (4, 2)])
def test_only_the_gradients_asked_for(device, monkeypatch, t, H, Hk):
    """The same bits as all of them, and the others' kernels are not launched."""
    from craft_amd import autograd
    q, k, v, go = make(t, 2, 150, 150, H, Hk, 64)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    want = torch.autograd.grad(autograd.attention(*leaves, causal=True), leaves, go)
    seen = calls_of(monkeypatch)
    for some in ((0,), (1,), (2,), (0, 2), (1, 2)):
        xs = [x.clone().requires_grad_(n in some) for n, x in enumerate((q, k, v))]
        got = torch.autograd.grad(autograd.attention(*xs, causal=True), [xs[n] for n in some], go)
        assert all(torch.equal(g, want[n]) for g, n in zip(got, some))
        name, args = seen[-1]
        assert name == "craft_attention_bwd" and [a is not None for a in args[17:20]] == [0 in some, some != (0,), some != (0,)]


def test_gradients_entry_point_takes_what_is_asked_for():
    import ctypes

    from craft_amd import hip
    lib, buf = hip.load(), 4096
    shape = (ctypes.c_long * 21)(*([1, 4, 4, 2, 2, 16] + [128, 32, 16] * 5))
    bwd = lambda dq, dk, dv, group=0: lib.craft_attention_bwd(buf, buf, buf, buf, None, buf, buf, shape, None, None, None, None, 1.0, 0.0, 0, 1, group, dq, dk, dv, buf, 1 << 20, None)  # noqa: E731
    assert bwd(None, None, None) == 0                                      # (nothing asked for: nothing launched)
    assert bwd(buf, None, buf) == 10001 and bwd(buf, buf, None) == 10001 and bwd(buf, None, None, 1) == 10001
    assert bwd(buf + 8, None, None) == 10002 and bwd(None, buf, buf + 8) == 10002


@pytest.mark.parametrize("dims, t, docs, want", [
    ((1, 16, 32768, 32, 8, 128), "bf16", False, 32), ((1, 17, 32768, 32, 8, 128), "bf16", False, 21), ((1, 256, 32768, 32, 8, 128), "bf16", False, 2),
    ((1, 257, 32768, 32, 8, 128), "bf16", False, 0), ((1, 17, 32768, 32, 8, 128), "bf16", True, 0), ((1, 16, 32768, 32, 8, 128), "bf16", True, 32),
    ((1, 17, 2047, 32, 8, 128), "fp16", False, 0), ((1, 17, 2048, 32, 8, 128), "fp16", False, 8), ((1, 17, 511, 32, 8, 64), "fp32", False, 0),
    ((1, 17, 512, 32, 8, 64), "fp32", False, 2), ((1, 1, 4096, 128, 1, 128), "bf16", False, 16), ((16, 1, 32768, 32, 8, 128), "bf16", False, 4),
    ((700, 1, 10, 1, 1, 64), "fp32", False, 1), ((1, 1, 1, 1, 1, 8), "bf16", False, 1)])
def test_which_kernel(dims, t, docs, want):
    """Few rows, and more of them where the keys are long and split in two at least, take the kernel whose keys are split."""
    from craft_amd import ops
    plan = object.__new__(ops.AttentionPlan)
    plan.dims, plan.code, plan.docs = dims, ops.DTYPE_CODE[TYPES[t]], torch.zeros(1) if docs else None
    assert plan.splits() == want


@gpu
@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("shape, how", [
    ((1, 17, 2100, 16, 4, 128), dict(causal=True)), ((1, 33, 2048, 8, 2, 64), dict(causal=True, cap=10.0)), ((2, 100, 3001, 6, 2, 72), dict(causal=True, slopes=True)),
    ((1, 1, 2500, 128, 1, 64), dict(causal=True)), ((1, 130, 2050, 3, 3, 32), {}), ((3, 90, 2111, 2, 2, 40), dict(causal=True, prefix=[1990, 0, 2111])),
    ((1, 2049, 2049, 1, 1, 64), dict(causal=True)), ((1, 2300, 2060, 2, 2, 24), dict(causal=True, cap=5.0, slopes=True))])
def test_a_chunk_against_long_keys(device, t, shape, how):
    """More than 64 rows with their keys split: whole prompts, rows that see nothing (more queries than keys), many heads on one key head."""
    from craft_amd import ops
    B, nq, nk, H, Hk, D = shape
    how = dict(how)
    if how.get("slopes"):
        how["slopes"] = slopes_of(H)
    if "prefix" in how:
        how["prefix"] = torch.tensor(how["prefix"], dtype=torch.int32, device="cuda")
    q, k, v, _ = make(t, *shape)
    assert ops.AttentionPlan(q, k, v, None, 0.0, None, False, None, None, None).splits() >= 2 and nq * H // Hk > 64
    res, tol = attention64(q, k, v, **how)
    check([ops.attention(q, k, v, **how)], res, tol)


@gpu
@pytest.mark.parametrize("B, n, H, Hk, D", [(1000, 33, 4, 4, 40), (1, 40000, 2, 1, 72), (3, 2050, 8, 1, 64)])
def test_norms_of_many_and_long_rows(device, B, n, H, Hk, D):
    """The largest norms of fp16's gradients over many short rows and over more slices than there are: the score gradients of the rows that hold them
    pass fp16's range without a scale.  Against the same arithmetic in fp32: off by the result's rounding and, in the mean, by one operand's (u = 2^-11; few
    terms stand out here, so that it does not average out)."""
    from craft_amd import autograd
    q, k, v, go = make("fp16", B, n, n, H, Hk, D, spread=0.5)
    go *= 1e-4
    go[-1, n - 7, H - 1], v[-1, n - 9, Hk - 1] = 200.0, 100.0
    how = dict(causal=True) if n < 10000 else dict(docs=(torch.arange(n, dtype=torch.int32, device="cuda") // 200)[None])
    leaves = [x.requires_grad_() for x in (q, k, v)]
    got = torch.autograd.grad(autograd.attention(*leaves, **how), leaves, go)
    wide = [x.detach().float().requires_grad_() for x in (q, k, v)]
    want = torch.autograd.grad(autograd.attention(*wide, **how), wide, go.float())
    for g, w, name in zip(got, want, ("dq", "dk", "dv")):
        assert torch.isfinite(g).all(), name
        off, least = (g.double() - w.double()).norm().item(), unavoidable(w.double(), torch.float16)
        assert off <= least + 2.0 ** -11 * w.double().norm().item(), (name, off / least)


def test_memory_that_is_shared_or_not():
    from craft_amd import ops
    flat = torch.zeros(4096)
    at = lambda o, shape, strides: torch.as_strided(flat, shape, strides, o)                  # noqa: E731
    a, b, c = torch.zeros(2, 5, 3, 4, 8).unbind(2)
    assert ops._apart(a, b) and ops._apart(b, a) and ops._apart(a, c) and not ops._apart(a, a)            # slices of one projection
    a, b, c = torch.zeros(2, 5, 4, 3, 8).unbind(3)                                            # within a head
    assert ops._apart(a, b) and ops._apart(c, a)
    x = torch.zeros(3, 20, 2, 8)
    assert ops._apart(x[:, :5], x[:, 5:9]) and not ops._apart(x[:, :5], x[:, 4:9]) and ops._apart(x[:1], x[1:2]) and not ops._apart(x[:2], x[1:])
    assert ops._apart(x[..., :4], x[..., 4:]) and not ops._apart(x[..., :5], x[..., 4:]) and ops._apart(flat[:10], flat[10:]) and not ops._apart(flat[:10], flat[9:])
    assert not ops._apart(flat[:8].expand(6, 8), flat[:48].view(6, 8)) and not ops._apart(at(0, (4, 8), (10, 1)), at(6, (4, 8), (10, 1)))
    # (against every element, over random pairs: what it calls apart is)
    g = torch.Generator().manual_seed(0)
    r = lambda hi: int(torch.randint(0, hi, (1,), generator=g))                               # noqa: E731
    proven = 0
    for _ in range(400):
        t = [at(r(60), (1 + r(3), 1 + r(4), 1 + r(5)), (r(4) * 12, r(3) * 6, 1 + r(2))) for _ in range(2)]
        places = [{o + i * s[0] + j * s[1] + k * s[2] for i in range(n[0]) for j in range(n[1]) for k in range(n[2])}
                  for o, s, n in ((y.storage_offset(), y.stride(), y.shape) for y in t)]
        if ops._apart(*t):
            proven += 1
            assert not places[0] & places[1]
        for y, p in zip(t, places):
            assert not ops._owns_its_elements(y) or len(p) == y.numel()
    assert proven > 40


@gpu
@pytest.mark.parametrize("nq", [1, 40])
def test_out_that_shares_memory(device, nq):
    """q's own memory and slices beside q, k and v are written; what overlaps them is refused."""
    from craft_amd import ops
    from craft_amd.hip import CraftHipError
    g = torch.Generator().manual_seed(4)
    qkvo = torch.randn(2, 60, 4, 2, 64, generator=g).bfloat16().cuda()
    q, k, v, o = qkvo.unbind(2)
    want = ops.attention(q[:, :nq], k, v)
    assert torch.equal(ops.attention(q[:, :nq], k, v, out=o[:, :nq]), want) and torch.equal(o[:, :nq], want)
    later = q[:, nq:2 * nq] if 2 * nq <= 60 else q[:, :0]
    assert later.numel() == 0 or torch.equal(ops.attention(q[:, :nq], k, v, out=later), want)
    for bad in (k[:, :nq], v[:, :nq], v[:, 1:nq + 1], q[:, 1:nq + 1] if nq > 1 else k[:, 5:6], qkvo[:, :nq, 1:3].flatten(2, 3)[:, :, 1:3],
                torch.as_strided(qkvo, (2, nq, 2, 64), (0, 512, 64, 1)), torch.as_strided(o.clone(), (2, nq, 2, 64), (8, 128, 64, 1))):
        with pytest.raises(CraftHipError, match="out must"):
            ops.attention(q[:, :nq], k, v, out=bad)
    assert torch.equal(ops.attention(q[:, :nq], k, v, out=q[:, :nq]), want)


@gpu
@pytest.mark.parametrize("t", list(TYPES))
def test_captured_gradients(device, t):
    """A training step's forward and backward pass in a graph whose replays follow new inputs, eager steps between them; every replay against eager."""
    from craft_amd import autograd
    q, k, v, go = make(t, 2, 150, 150, 4, 2, 72)
    docs = doc_ids(2, 150, 4, 30)
    w = torch.ones(72, device="cuda").to(q.dtype)

    def step(q, k, v, go, w):
        leaves = [x.detach().requires_grad_() for x in (q, k, v, w)]
        o = autograd.layer_norm(autograd.attention(*leaves[:3], docs=docs, causal=True, cap=20.0), leaves[3])
        return [o, *torch.autograd.grad(o, leaves, go)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(q, k, v, go, w)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(q, k, v, go, w)
    for seed in range(4):
        for x, y in zip((q, k, v, go), make(t, 2, 150, 150, 4, 2, 72, seed=seed)):
            x.copy_(y * (1 if seed < 2 else 1e-4))
        docs.copy_(doc_ids(2, 150, 4, 30, seed=seed))
        graph.replay()
        torch.cuda.synchronize()
        want = step(q, k, v, go, w)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
