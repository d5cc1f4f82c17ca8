"""Attention with a cap, a distance bias and masks in 64 bits, with its gradients and, element by element, how far a kernel of a given type may be off."""
import math

import torch


def visible(nq, nk, causal=False, prefix=None, docs=None, docs_k=None, batch=1):
    i = torch.arange(nq)[:, None] + (nk - nq)
    j = torch.arange(nk)[None, :]
    see = torch.ones(batch, nq, nk, dtype=torch.bool) if not causal else (j <= i).expand(batch, nq, nk).clone()
    if prefix is not None:
        see |= j < prefix.cpu()[:, None, None]
    if docs is not None:
        dk = docs if docs_k is None else docs_k
        see &= (docs.cpu()[:, :, None] == dk.cpu()[:, None, :]) & (dk.cpu()[:, None, :] >= 0)
    return see


def attention64(q, k, v, go=None, scale=None, cap=0.0, slopes=None, causal=False, prefix=None, docs=None, docs_k=None):
    """(results, tolerances): o, and with ``go`` also dq, dk, dv.  The tolerance counts, with u half a step of the tensors' type: the final rounding, the
    rounding of the probabilities and score gradients to the type for the second products, the fp32 sums (as many roundings as terms), the rounded o
    inside delta, and what an error of a score does to its exponential."""
    t = q.dtype
    u, w = torch.finfo(t).eps / 2, 2.0 ** -24
    # A result below the type's smallest normal number is rounded to a multiple of its smallest step s, off by s / 2 whatever its size: for fp16 s = 2^-24
    # (2^-14 smallest normal x 2^-10), so 2^-25 = 2.98e-8 is added to every tolerance; a gradient of 3.32e-8 is stored as 5.96e-8, 2.64e-8 off, where u
    # times its value allows 1.6e-11.  (bf16 and fp32: s below 1e-40; 1e-30 stands for it.)
    tiny = 2.0 ** -25 if t == torch.float16 else 1e-30
    q, k, v = (x.detach().cpu().double() for x in (q, k, v))
    B, nq, H, D = q.shape
    nk, Hk = k.shape[1:3]
    G = H // Hk
    scale = D ** -0.5 if scale is None else scale
    see = visible(nq, nk, causal, prefix, docs, docs_k, B)[:, None]
    if docs is not None:                                                   # what padding holds does not count
        dk_ = docs if docs_k is None else docs_k
        q = torch.where((docs.cpu() < 0)[:, :, None, None], 0.0, q)
        k, v = (torch.where((dk_.cpu() < 0)[:, :, None, None], 0.0, x) for x in (k, v))
    q = q.transpose(1, 2)
    k, v = (x.transpose(1, 2).repeat_interleave(G, 1) for x in (k, v))
    raw = scale * q @ k.mT
    z = cap * torch.tanh(raw / cap) if cap else raw.clone()
    slope = 1 - torch.tanh(raw / cap) ** 2 if cap else torch.ones_like(raw)
    away = ((torch.arange(nq)[:, None] + (nk - nq)) - torch.arange(nk)[None, :]).abs().double()
    if slopes is not None:
        z = z - slopes.cpu().double()[:, None, None] * away
    # error of a score: D roundings of its products' sum, and a few of its own size (scaling, cap, bias, difference from the row's maximum)
    size = abs(scale) * (q.abs() @ k.abs().mT)
    ez = D * w * size + 8 * w * (z.abs() + z.masked_fill(~see, 0.0).abs().amax(-1, keepdim=True) + (cap or 0.0))
    if t != torch.float32 and cap:
        ez = ez + 4 * w * cap                                              # the quick tanh
    top = z.masked_fill(~see, -math.inf).amax(-1, keepdim=True)
    p = torch.where(see, torch.exp(z - torch.where(top.isinf(), 0.0, top)), 0.0)
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    ep = 2 * ez + (nk + 8) * w                                             # relative error of a probability (its own score's and the sum's)
    ep = torch.where(see, ep, 0.0)
    ep = ep + (p * ep).sum(-1, keepdim=True)
    o = p @ v
    to = u * o.abs() + (p * (u + ep)) @ v.abs() + nk * w * (p @ v.abs()) + tiny
    res, tol = [o.transpose(1, 2)], [to.transpose(1, 2)]
    if go is None:
        return res, tol
    go = go.detach().cpu().double()
    if docs is not None:
        go = torch.where((docs.cpu() < 0)[:, :, None, None], 0.0, go)
    go = go.transpose(1, 2)
    dv = p.mT @ go
    tv = (p * (u + ep)).mT @ go.abs() + nq * G * w * (p.mT @ go.abs())
    dp = go @ v.mT
    delta = (go * o).sum(-1, keepdim=True)
    ds = p * (dp - delta) * slope
    edp = D * w * (go.abs() @ v.abs().mT) + (go.abs() * to).sum(-1, keepdim=True) + D * w * (go.abs() * o.abs()).sum(-1, keepdim=True)
    # fp16: below its smallest normal number (2^-14) a score gradient keeps an absolute step only
    floor = 2.0 ** -25 if t == torch.float16 else 0.0
    eslope = 4 * ez / cap + 8 * w if cap else torch.zeros_like(ez)         # of 1 - tanh^2, absolutely
    eds = ds.abs() * (u + ep + 8 * w) + p * slope * edp + p * (dp - delta).abs() * eslope + floor * see
    dq = scale * ds @ k
    tq = abs(scale) * (eds @ k.abs()) + nk * w * abs(scale) * (ds.abs() @ k.abs())
    dk = scale * ds.mT @ q
    tk = abs(scale) * (eds.mT @ q.abs()) + nq * G * w * abs(scale) * (ds.abs().mT @ q.abs())
    fold = lambda x: x.unflatten(1, (Hk, G)).sum(2)                        # noqa: E731
    dk, dv, tk, tv = fold(dk), fold(dv), fold(tk), fold(tv)
    if t == torch.float16:
        tv = tv + nq * G * 2.0 ** -25 * go.abs().amax()                    # (probabilities below 2^-14 likewise)
    for r, e in ((dq, tq), (dk, tk), (dv, tv)):
        res.append(r.transpose(1, 2))
        tol.append((e + u * r.abs() + tiny).transpose(1, 2))
    return res, tol


def check(got, res, tol):
    for g, r, e, name in zip(got, res, tol, ("o", "dq", "dk", "dv")):
        assert g.shape == r.shape, (name, g.shape, r.shape)
        off = (g.detach().cpu().double() - r).abs()
        assert torch.isfinite(off).all(), f"{name}: not finite"
        worst = (off / e).max().item() if off.numel() else 0.0
        assert worst <= 1.0, f"{name}: {worst:.2f} times the bound, at most {off.max().item():.3g} off"
