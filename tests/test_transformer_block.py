"""The operators as one training step uses them: a pre-norm attention block (layer norm, projections, attention over packed sequences with padding, residual),
its gradients against the same block in 64 bits, one Muon step on its weights, and its tokens one by one against the whole."""
import pytest
import torch

from attention_reference import visible
from test_orthogonalize import iterate

gpu = pytest.mark.gpu
H, HK, D, C = 4, 2, 32, 96


class Block(torch.nn.Module):
    """x + proj(attention(norm(x))) with this package's operators where ``own`` is true, with torch's elementary ones otherwise."""

    def __init__(self, own):
        super().__init__()
        self.own = own
        self.weight, self.bias = torch.nn.Parameter(torch.ones(C)), torch.nn.Parameter(torch.zeros(C))
        self.q, self.kv, self.out = torch.nn.Linear(C, H * D, bias=False), torch.nn.Linear(C, 2 * HK * D, bias=False), torch.nn.Linear(H * D, C)

    def heads(self, y):
        B, N = y.shape[:2]
        k, v = self.kv(y).view(B, N, 2, HK, D).unbind(2)                   # (views of one projection: read in place)
        return self.q(y).view(B, N, H, D), k, v

    def forward(self, x, docs, cap, slopes):
        from craft_amd import autograd
        B, N = x.shape[:2]
        if self.own:
            q, k, v = self.heads(autograd.layer_norm(x, self.weight, self.bias))
            o = autograd.attention(q, k, v, cap=cap, slopes=slopes, causal=True, docs=docs)
        else:
            q, k, v = (t.transpose(1, 2) for t in self.heads(torch.nn.functional.layer_norm(x, (C,), self.weight, self.bias, 1e-5)))
            k, v = (t.repeat_interleave(H // HK, 1) for t in (k, v))
            z = cap * torch.tanh(q @ k.mT / D ** 0.5 / cap)
            i = torch.arange(N, device=x.device)
            z = z - slopes.to(x.dtype)[:, None, None] * (i[:, None] - i).abs()
            see = visible(N, N, True, docs=docs, batch=B)[:, None].to(x.device)
            o = (torch.softmax(z.masked_fill(~see, -1e30), -1) * see.any(-1, keepdim=True) @ v).transpose(1, 2)
        return x + self.out(o.reshape(B, N, H * D))


def pair(seed=0):
    torch.manual_seed(seed)
    own, ref = Block(True), Block(False)
    with torch.no_grad():
        for p in own.parameters():
            if p.dim() > 1:
                p.normal_(0, p.shape[1] ** -0.5)
            else:
                p.add_(0.1 * torch.randn(p.shape))
    ref.load_state_dict(own.state_dict())
    return own.cuda(), ref.double().cuda()


def data(seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(2, 75, C, generator=g).cuda()
    docs = torch.full((2, 75), -1, dtype=torch.int32)
    docs[0, :20], docs[0, 20:61], docs[1, :75] = 0, 1, 4
    go = torch.randn(2, 75, C, generator=g).cuda()
    return x, docs.cuda(), go, torch.tensor([0.5, 0.25, 0.1, 0.0], device="cuda")


@gpu
def test_gradients_of_the_block(device):
    """fp32: every sum of the block is of at most 1 000 terms of unit size, so a gradient is off by a few hundred times 2^-24 of its size: 5e-5."""
    own, ref = pair()
    x, docs, go, slopes = data()
    x1, x2 = x.clone().requires_grad_(), x.double().requires_grad_()
    y1, y2 = own(x1, docs, 5.0, slopes), ref(x2, docs, 5.0, slopes)
    assert (y1.double() - y2).norm() < 5e-5 * y2.norm()
    g1 = torch.autograd.grad(y1, [x1, *own.parameters()], go)
    g2 = torch.autograd.grad(y2, [x2, *ref.parameters()], go.double())
    for a, b in zip(g1, g2):
        assert (a.double() - b).norm() < 5e-5 * b.norm() + 1e-7


@gpu
def test_a_muon_step_of_the_block(device):
    """backward() into FlatMuon's flat gradients and one step: the three weight matrices by the orthogonalised gradient (the first step's Nesterov momentum is
    1 + mu times the gradient, which the norm takes out), to what the gradients' own error of 5e-5 (see above) becomes
    in the iteration."""
    from craft_amd.train import FlatMuon
    own, ref = pair()
    x, docs, go, slopes = data()
    opt = FlatMuon(own.parameters(), lr=0.1, weight_decay=0.0)
    before = {k: p.detach().clone() for k, p in own.named_parameters()}
    opt.zero_grad()
    own(x, docs, 5.0, slopes).backward(go)
    opt.step()
    names = [k for k, _ in own.named_parameters()]
    assert [names[i] for i in opt.matrix_index] == ["q.weight", "kv.weight", "out.weight"]
    grads = dict(zip((k for k, _ in ref.named_parameters()), torch.autograd.grad(ref(x.double(), docs, 5.0, slopes), list(ref.parameters()), go.double())))
    for k in ("q.weight", "kv.weight", "out.weight"):
        o, _ = iterate(grads[k])
        step = 0.1 * 0.2 * max(o.shape) ** 0.5 * o
        moved = (before[k].double() - own.get_parameter(k).double()).cpu()
        # (the polynomial multiplies small singular directions of the gradient by up to 3.4445^5 = 485, and their errors with them: 485 * 5e-5 = 2.4e-2 at most)
        assert (moved - step).norm() < 2e-2 * step.norm(), k


@gpu
def test_tokens_one_by_one(device):
    """Serving: each new token against a growing cache gives the row that the whole sequence gives (the single-token kernel against the block kernel)."""
    from craft_amd import ops
    own, _ = pair()
    x, _, _, slopes = data()
    with torch.no_grad():
        q, k, v = own.heads(ops.layer_norm(x, own.weight, own.bias))
        whole = ops.attention(q, k, v, cap=5.0, slopes=slopes, causal=True)
        cache = [torch.zeros(2, 80, HK, D, device="cuda") for _ in range(2)]
        for n in range(75):
            y = ops.layer_norm(x[:, n:n + 1], own.weight, own.bias)
            a, b, c = own.heads(y)
            cache[0][:, n:n + 1], cache[1][:, n:n + 1] = b, c
            one = ops.attention(a, cache[0][:, :n + 1], cache[1][:, :n + 1], cap=5.0, slopes=slopes, causal=True)
            # fp32 on both sides: projections of one row and of many differ by their sums' order, 96 roundings of unit values
            assert (one - whole[:, n:n + 1]).abs().max() < 2e-5, n


@gpu
def test_the_documented_calls_run(device):
    """The documented example (the integration guide's last section) as it stands: its single token gives its row of the whole attention."""
    import os
    import re
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "INTEGRATION.md")).read()
    ns = {}
    exec(re.search(r"```python\n(.*?)```", text[text.index("## 4."):], flags=re.S).group(1), ns)      # noqa: S102 -- our own document
    # fp32 on both sides, sums of at most 100 unit values in another order
    assert (ns["one"] - ns["o"].detach()[:, 89:90]).abs().max() < 2e-5
    assert torch.isfinite(ns["proj"].weight).all()
