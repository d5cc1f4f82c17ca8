"""The cases at which the layer norm, the masked and biased attention and the orthogonalisation of updates are measured.

``listed()`` names the cases, ``draw`` gives more of the same ranges, ``prepare`` makes a case's inputs on the GPU, ``run`` is one pass.
Where ``own`` is false a pass is elementary torch arithmetic in 32 bits, rounded once at the end; where it is true it is the calls that a user
makes of ``craft_amd``.  ``exact`` computes the same outputs in 64 bits from the definitions."""
import math

import torch

own = False

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}

#: rows x columns (x how many) of every weight of the CRAFT model (f2 full, setrans) that is a matrix with at least 16 rows and columns once a
#: convolution's kernel window is flattened into its columns
MODEL = ("64x147x2,64x576x8,64x1152x1,96x64x2,96x576x2,96x864x6,126x2304x1,128x96x2,128x98x1,128x128x2,128x864x2,128x1152x6,128x2560x6,192x2304x1,"
         "256x128x2,256x256x3,256x324x1,256x1152x2,512x128x1,576x256x1,1024x256x1")


def listed():
    norm = {"op": "layer_norm", "train": True, "affine": "same"}
    attn = {"op": "attention", "causal": False, "prefix": 0, "docs": 0, "padding": 0, "cap": 0.0, "slopes": False, "train": False}
    return [
        # the tokens of four 448 x 1024 frames at 1/8 of their size, normalised as every transformer of the model does, inference
        dict(norm, name="norm_tokens", type="fp32", rows=28672, width=256, train=False, affine="fp32"),
        # a training step of a wide model: 16 k tokens, bf16 activations and weights, all three gradients
        dict(norm, name="norm_wide_train", type="bf16", rows=16384, width=4096),
        # an odd batch of odd rows that no vector load fits, fp32 weights beside fp16 activations
        dict(norm, name="norm_odd_train", type="fp16", rows=1441, width=1027, affine="fp32"),
        # a training step of a causal model whose scores are capped, four query heads to a key head
        dict(attn, name="attn_capped_train", type="bf16", batch=2, queries=4096, keys=4096, heads=16, kv_heads=4, width=128, causal=True, cap=30.0, train=True),
        # self-attention among the tokens of a 368 x 496 training crop (46 x 62 at 1/8), 4 modes of 64, scores falling with the distance, fp32
        dict(attn, name="attn_bias_train_fp32", type="fp32", batch=2, queries=2852, keys=2852, heads=4, kv_heads=4, width=64, slopes=True, train=True),
        # several images of unequal size packed into each row of a batch, with padding behind them: nothing crosses an image's border
        dict(attn, name="attn_packed_train", type="fp16", batch=4, queries=3001, keys=3001, heads=8, kv_heads=8, width=64, docs=7, padding=173, train=True),
        # a long prompt whose first tokens are seen by all
        dict(attn, name="attn_prefix_prompt", type="fp16", batch=1, queries=8192, keys=8192, heads=32, kv_heads=8, width=128, causal=True, prefix=1900),
        # one new token for each of 16 sequences against long caches
        dict(attn, name="attn_token_long", type="bf16", batch=16, queries=1, keys=32768, heads=32, kv_heads=8, width=128, causal=True, cap=30.0),
        # one new token of one sequence with a short cache: latency
        dict(attn, name="attn_token_short", type="fp16", batch=1, queries=1, keys=777, heads=8, kv_heads=8, width=64, causal=True, slopes=True),
        # the update of one training step of the model: every matrix of it
        {"op": "orthogonalize", "name": "update_model", "shapes": MODEL},
        # one square projection: latency
        {"op": "orthogonalize", "name": "update_small", "shapes": "256x256x1"},
        # the feed-forward matrix of a wide model
        {"op": "orthogonalize", "name": "update_wide", "shapes": "2048x8192x1"},
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm, odd as often as even."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


#: no drawn case does more than the largest listed ones (operations of 16-bit and of fp32 cases, bytes)
MOST = {"fp16": 550e9, "bf16": 550e9, "fp32": 90e9, "bytes": 2.1e9}


def draw(rng):
    c = _draw(rng)
    while work(c)["flops"] > MOST[c.get("type", "bf16")] or work(c)["bytes"] > MOST["bytes"]:
        c = _draw(rng)
    return c


def _draw(rng):
    op = rng.choice(["layer_norm", "attention", "attention", "attention", "orthogonalize"])
    if op == "layer_norm":
        width = _log(rng, 17, 8192)
        return {"op": op, "train": rng.random() < 0.6, "affine": rng.choice(["same", "fp32"]), "type": rng.choice(list(TYPES)),
                "rows": _log(rng, 1, (16384 * 4096) // width), "width": width}
    if op == "orthogonalize":
        if rng.random() < 0.5:
            return {"op": op, "shapes": "%dx%dx1" % (_log(rng, 16, 1500), _log(rng, 16, 4500))}
        return {"op": op, "shapes": ",".join("%dx%dx%d" % (_log(rng, 16, 600), _log(rng, 16, 1500), rng.randint(1, 4)) for _ in range(rng.randint(2, 9)))}
    kind = rng.choice(["train", "train", "prompt", "token"])
    kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 1, 2, 3, 4])
    c = {"op": op, "type": rng.choice(["fp16", "bf16", "fp16", "bf16", "fp32"]), "heads": kv_heads * group, "kv_heads": kv_heads,
         "width": rng.choice([32, 40, 64, 64, 72, 128, 128]), "cap": rng.choice([0.0, 0.0, 15.0, 30.0, 50.0]), "slopes": rng.random() < 0.4, "train": kind == "train",
         "causal": True, "prefix": 0, "docs": 0, "padding": 0}
    if kind == "token":
        return dict(c, batch=_log(rng, 1, 16), queries=rng.choice([1, 1, 1, 2, 5]), keys=_log(rng, 5, 32768))
    n = _log(rng, 33, 4096)
    c.update(batch=rng.randint(1, 2) if n > 1500 else rng.randint(1, 6), queries=n, keys=n, causal=rng.random() < 0.6)
    if kind == "prompt" and rng.random() < 0.5:                      # a chunk of a prompt behind a cache
        c.update(keys=n + _log(rng, 1, 2000), causal=True)
    mask = rng.choice(["", "docs", "prefix"])
    if mask == "docs" and c["keys"] == n:
        c.update(docs=rng.randint(1, 9), padding=rng.choice([0, 1, n // 9]))
    if mask == "prefix":
        c.update(causal=True, prefix=rng.randint(1, n))
    return c


# ----------------------------------------------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------------------------------------------
def _shapes(case):
    return [(int(r), int(c)) for r, c, n in (s.split("x") for s in case["shapes"].split(",")) for _ in range(int(n))]


def _doc_lengths(case):
    """Unequal lengths of the packed pieces of every row of the batch (not of the seed: the work of a case is fixed)."""
    n, out = case["keys"] - case["padding"], []
    for b in range(case["batch"]):
        cut = sorted({int(n * ((0.6180339887 * (k + 1) + 0.11 * b) % 1.0)) for k in range(case["docs"] - 1)} | {0, n})
        out.append([q - p for p, q in zip(cut, cut[1:])])
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    if case["op"] == "layer_norm":
        t = TYPES[case["type"]]
        wt = t if case["affine"] == "same" else torch.float32
        rows, width = case["rows"], case["width"]
        # activations with an offset and a spread of their own in every row and a few channels far larger than the rest
        x = normal(rows, width) * (0.5 + normal(rows, 1).abs()) + 0.3 * normal(rows, 1)
        x[:, ::97] *= 6.0
        s = {"x": x.to(t), "w": (1.0 + 0.2 * normal(width)).to(wt), "b": (0.1 * normal(width)).to(wt), "train": case["train"]}
        if case["train"]:
            for k in "xwb":
                s[k].requires_grad_()
            s["dy"] = normal(rows, width).to(t)
        return dict(s, op=case["op"])
    if case["op"] == "orthogonalize":
        mats = []
        for m, n in _shapes(case):
            # a gradient: a sum of strong directions over many weak ones, of a gradient's size
            r = max(1, min(m, n) // 8)
            mats.append((normal(m, r) @ normal(r, n) / r ** 0.5 + 0.3 * normal(m, n)) * 1e-3)
        return {"op": case["op"], "mats": mats}
    t = TYPES[case["type"]]
    B, Nq, Nk, H, Hk, D = (case[k] for k in ("batch", "queries", "keys", "heads", "kv_heads", "width"))
    # scores of a spread of about 3: some keys stand out of a row, none takes all of it
    s = {"q": (3.0 * normal(B, Nq, H, D)).to(t), "k": normal(B, Nk, Hk, D).to(t), "v": normal(B, Nk, Hk, D).to(t), "causal": case["causal"], "cap": case["cap"],
         "train": case["train"], "slopes": None, "prefix": None, "docs": None}
    if case["train"]:
        for k in "qkv":
            s[k].requires_grad_()
        s["do"] = normal(B, Nq, H, D).to(t)
    if case["slopes"]:
        s["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device="cuda")
    if case["prefix"]:
        s["prefix"] = torch.tensor([max(1, case["prefix"] - 3 * b) for b in range(B)], device="cuda", dtype=torch.int32)
    if case["docs"]:
        ids = torch.full((B, Nk), -1, dtype=torch.int32)
        for b, lengths in enumerate(_doc_lengths(case)):
            ids[b, :sum(lengths)] = torch.repeat_interleave(torch.arange(len(lengths), dtype=torch.int32), torch.tensor(lengths))
        s["docs"] = ids.cuda()
    return dict(s, op=case["op"])


# ----------------------------------------------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------------------------------------------
def _run_own(s):
    from craft_amd import autograd, ops
    if s["op"] == "layer_norm":
        if not s["train"]:
            return ops.layer_norm(s["x"], s["w"], s["b"])
        y = autograd.layer_norm(s["x"], s["w"], s["b"])
        return [y, *torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])]
    if s["op"] == "orthogonalize":
        return ops.orthogonalize(s["mats"])
    how = dict(cap=s["cap"], slopes=s["slopes"], causal=s["causal"], prefix=s["prefix"], docs=s["docs"])
    if not s["train"]:
        return ops.attention(s["q"], s["k"], s["v"], **how)
    o = autograd.attention(s["q"], s["k"], s["v"], **how)
    return [o, *torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])]


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"layer_norm": _norm, "attention": _attention, "orthogonalize": _orthogonalize}[state["op"]](state)


def _norm(s):
    x, w = s["x"].float(), s["w"].float()
    mean = x.mean(-1, keepdim=True)
    rstd = ((x - mean).square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    xn = (x - mean) * rstd
    y = (xn * w + s["b"].float()).to(s["x"].dtype)
    if not s["train"]:
        return y
    dy = s["dy"].float()
    dxn = dy * w
    dx = (dxn - dxn.mean(-1, keepdim=True) - xn * (dxn * xn).mean(-1, keepdim=True)) * rstd
    return [y, dx.to(s["x"].dtype), (dy * xn).sum(0).to(s["w"].dtype), dy.sum(0).to(s["b"].dtype)]


def _visible(s, nq, nk, device):
    """[B or 1, 1, nq, nk]: which keys a query sees; a query's position is its index counted from the end of the keys."""
    i = torch.arange(nq, device=device)[:, None] + (nk - nq)
    j = torch.arange(nk, device=device)[None, :]
    see = (j <= i) if s["causal"] else torch.ones(nq, nk, device=device, dtype=torch.bool)
    see = see[None, None]
    if s["prefix"] is not None:
        see = see | (j < s["prefix"][:, None, None, None])
    if s["docs"] is not None:
        d = s["docs"]
        see = see & (d[:, None, :, None] == d[:, None, None, :]) & (d[:, None, None, :] >= 0)
    return see


def _attention(s):
    q, k, v = (s[n].float().transpose(1, 2) for n in "qkv")                       # [B, heads, N, D]
    H, Hk, nq, nk, D = q.shape[1], k.shape[1], q.shape[2], k.shape[2], q.shape[3]
    k, v = (t.repeat_interleave(H // Hk, 1).contiguous() for t in (k, v))
    scale = D ** -0.5
    x = (q.contiguous() @ k.transpose(2, 3).contiguous()).mul_(scale)
    slope = None
    if s["cap"]:
        x = x.div_(s["cap"]).tanh_()
        slope = 1.0 - x.square() if s["train"] else None
        x = x.mul_(s["cap"])
    if s["slopes"] is not None:
        i = torch.arange(nq, device=x.device)[:, None] + (nk - nq)
        x = x.sub_(s["slopes"][:, None, None] * (i - torch.arange(nk, device=x.device)[None, :]).abs())
    see = _visible(s, nq, nk, x.device)
    x = x.masked_fill_(~see, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = x.sub_(torch.where(top.isinf(), 0.0, top)).exp_()                          # a row that sees nothing: all zero
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total == 0, 1.0, total))
    o = (p @ v).transpose(1, 2).to(s["q"].dtype)
    if not s["train"]:
        return o
    do = s["do"].float().transpose(1, 2).contiguous()
    dv = p.transpose(2, 3).contiguous() @ do
    dp = do @ v.transpose(2, 3).contiguous()
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
    if slope is not None:
        ds = ds * slope
    dq = ds @ k
    dk = ds.transpose(2, 3).contiguous() @ q
    dk, dv = (t.unflatten(1, (Hk, H // Hk)).sum(2).transpose(1, 2).to(s["q"].dtype) for t in (dk, dv))
    return [o, dq.transpose(1, 2).to(s["q"].dtype), dk, dv]


def _orthogonalize(s):
    out = []
    for g in s["mats"]:
        x = (g.T if g.shape[0] > g.shape[1] else g)
        # (the norm in 64 bits: its error would scale the whole result)
        x = x / (x.double().square().sum().sqrt() + 1e-7).float()
        for _ in range(5):
            a = x @ x.T
            x = 3.4445 * x + (-4.7750 * a + 2.0315 * (a @ a)) @ x
        out.append(x.T.contiguous() if g.shape[0] > g.shape[1] else x)
    return out


# ----------------------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without, and its exact outputs
# ----------------------------------------------------------------------------------------------------------------------------------
def _pairs(case):
    """Visible (query, key) pairs of one head over the batch."""
    nq, nk, B = case["queries"], case["keys"], case["batch"]
    if case["docs"]:
        return sum((n * (n + 1) // 2 if case["causal"] else n * n) for lengths in _doc_lengths(case) for n in lengths)
    if not case["causal"]:
        return B * nq * nk
    off, total = nk - nq, 0
    for b in range(B):
        p = max(1, case["prefix"] - 3 * b) if case["prefix"] else 0
        below = max(0, min(nq, p - off))                              # queries that see the prefix and nothing behind it
        total += below * p + (nq - below) * off + (nq * (nq + 1) - below * (below + 1)) // 2
    return total


def work(case):
    if case["op"] == "orthogonalize":
        sizes = [(min(s), max(s)) for s in _shapes(case)]
        # a step: X X^T and its square (both symmetric: half a product each) and the product with X
        return {"bytes": 8 * sum(m * n for m, n in sizes), "flops": 5 * sum(m * (m + 1) * n + m * m * (m + 1) + 2 * m * m * n for m, n in sizes)}
    size = 4 if case["type"] == "fp32" else 2
    if case["op"] == "layer_norm":
        n, wsize = case["rows"] * case["width"], 4 if case["affine"] == "fp32" else size
        return {"bytes": n * size * (4 if case["train"] else 2) + case["width"] * wsize * (4 if case["train"] else 2), "flops": n * (20 if case["train"] else 8)}
    rows_q = case["batch"] * case["queries"] * case["heads"] * case["width"]
    rows_k = case["batch"] * case["keys"] * case["kv_heads"] * case["width"]
    # forward: q, k, v, o; with the gradients also do, dq, dk, dv
    return {"bytes": size * (rows_q * (4 if case["train"] else 2) + rows_k * (4 if case["train"] else 2)),
            "flops": _pairs(case) * case["heads"] * case["width"] * (14 if case["train"] else 4)}


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "layer_norm":
        x, w, b = (s[k].detach().double().requires_grad_() for k in "xwb")
        c = x - x.sum(-1, keepdim=True) / x.shape[-1]
        y = c / ((c * c).sum(-1, keepdim=True) / x.shape[-1] + 1e-5).sqrt() * w + b
        if not s["train"]:
            return y.detach()
        return [y.detach(), *torch.autograd.grad(y, (x, w, b), s["dy"].double())]
    if s["op"] == "orthogonalize":
        out = []
        for g in s["mats"]:
            y = g.double()
            y = y / (torch.linalg.vector_norm(y) + 1e-7)
            for _ in range(5):                                         # from the smaller side, whichever it is
                if y.shape[0] <= y.shape[1]:
                    a = y @ y.mT
                    y = 3.4445 * y - 4.7750 * (a @ y) + 2.0315 * (a @ (a @ y))
                else:
                    a = y.mT @ y
                    y = 3.4445 * y - 4.7750 * (y @ a) + 2.0315 * ((y @ a) @ a)
            out.append(y)
        return out
    B, nq, H, D = s["q"].shape
    nk, Hk = s["k"].shape[1:3]
    see = _visible(s, nq, nk, "cuda")
    away = (torch.arange(nk - nq, nk, device="cuda")[:, None] - torch.arange(nk, device="cuda")).abs().double()
    o = torch.zeros(B, nq, H, D, device="cuda", dtype=torch.float64)
    grads = [torch.zeros(t.shape, device="cuda", dtype=torch.float64) for t in (s["q"], s["k"], s["v"])] if s["train"] else []
    for b in range(B):
        m = see[min(b, see.shape[0] - 1), 0]
        some = m.any(-1, keepdim=True)
        for h in range(H):
            q, k, v = (t.detach().double().requires_grad_(s["train"]) for t in (s["q"][b, :, h], s["k"][b, :, h // (H // Hk)], s["v"][b, :, h // (H // Hk)]))
            z = q @ k.mT / math.sqrt(D)
            if s["cap"]:
                z = s["cap"] * torch.tanh(z / s["cap"])
            if s["slopes"] is not None:
                z = z - s["slopes"][h].double() * away
            z = torch.where(m, z, torch.where(some, -math.inf, 0.0))
            r = torch.exp(z - torch.logsumexp(z, -1, keepdim=True)) @ v * some
            o[b, :, h] = r.detach()
            if grads:
                for at, d in zip((grads[0][b, :, h], grads[1][b, :, h // (H // Hk)], grads[2][b, :, h // (H // Hk)]),
                                 torch.autograd.grad(r, (q, k, v), s["do"][b, :, h].double())):
                    at += d
    return [o, *grads] if grads else o
