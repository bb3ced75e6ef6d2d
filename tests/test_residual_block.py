"""The three operators as a model uses them: blocks of residual_norm and linear_act trained by FusedAdamW, eagerly and as one hipGraph,
and the single-row form of the same block."""
import copy

import pytest
import torch

import gcpnet_amd as G
from gcpnet_amd.graphs import GraphedStep

EPS32 = 2.0 ** -24


class Block(torch.nn.Module):
    """h = pre(s); s' = s + 0.5 * sigmoid(gate) * post(down(silu(up(h)))), the norms of two blocks' border in one call."""

    def __init__(self, d, wide, dtype):
        super().__init__()
        new = lambda *s, std=1.0: torch.nn.Parameter((torch.randn(*s) * std).to(dtype))  # noqa: E731
        self.up, self.up_b = new(wide, d, std=d ** -0.5), new(wide, std=0.1)
        self.down, self.down_b = new(d, wide, std=wide ** -0.5), new(d, std=0.1)
        self.gate, self.post = new(d), torch.nn.Parameter(torch.ones(d, dtype=dtype))
        self.pre, self.pre_b = torch.nn.Parameter(torch.ones(d, dtype=dtype)), torch.nn.Parameter(torch.zeros(d, dtype=dtype))

    def forward(self, s, h):
        y = G.linear_act(G.linear_act(h, self.up, self.up_b, act="silu"), self.down, self.down_b, residual=h)
        return G.residual_norm(s, y, self.gate, scale=0.5, gate_act="sigmoid", post="rms", post_weight=self.post, pre="layer", pre_weight=self.pre,
                               pre_bias=self.pre_b)

    def plain(self, s, h):
        up = h @ self.up.t() + self.up_b
        y = (up * torch.sigmoid(up)) @ self.down.t() + self.down_b + h
        y = y / (y.square().mean(-1, keepdim=True) + 1e-5).sqrt() * self.post
        s = s + 0.5 * torch.sigmoid(self.gate) * y
        return s, torch.nn.functional.layer_norm(s, s.shape[-1:], self.pre, self.pre_b, 1e-5)


class Stack(torch.nn.Module):
    def __init__(self, layers=2, d=64, wide=160, dtype=torch.float32, seed=0):
        super().__init__()
        torch.manual_seed(seed)
        self.blocks = torch.nn.ModuleList(Block(d, wide, dtype) for _ in range(layers))

    def forward(self, x, plain=False):
        s, h = x, torch.nn.functional.layer_norm(x, x.shape[-1:], eps=1e-5) if plain else G.residual_norm(x, pre="layer")[1]
        for b in self.blocks:
            s, h = b.plain(s, h) if plain else b(s, h)
        return s, h


def loss_of(s, h, target):
    return ((h - target).square().mean() + 0.1 * s.square().mean()).float()


def data(rows, d, dtype, seed=1):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(rows, d, generator=g).to(dtype), torch.randn(rows, d, generator=g).to(dtype)


@pytest.mark.gpu
def test_gradients_of_a_stack():
    """Values and gradients of two blocks against 64 bits: every sum has at most 160 terms, and some 20 operations lie between a weight and
    the loss, each off by at most (160 + 24) half steps of the largest magnitude in its row or column, a few units: 2e-4 of the
    tensor's largest value is 20 * 184 * 2^-24."""
    model = Stack().cuda()
    twin = copy.deepcopy(model).cpu().double()
    x, target = data(50, 64, torch.float32)
    gx = x.cuda().requires_grad_()
    loss = loss_of(*model(gx), target.cuda())
    loss.backward()
    cx = x.double().requires_grad_()
    want = loss_of(*twin(cx, plain=True), target.double())
    want.backward()
    assert abs(loss.item() - want.item()) < 2.2e-4 * abs(want.item())
    pairs = [(gx.grad, cx.grad)] + [(p.grad, q.grad) for p, q in zip(model.parameters(), twin.parameters())]
    for k, (a, b) in enumerate(pairs):
        assert (a.cpu().double() - b).abs().max() <= 2.2e-4 * b.abs().max(), k


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,bits", [(torch.float32, 32), (torch.float32, 8), (torch.bfloat16, 32), (torch.bfloat16, 8)])
def test_training_runs_eagerly_and_as_a_graph(dtype, bits):
    """Eight steps (forward, backward, clipped AdamW) eagerly, and three eager steps with five replays: the same parameters, bit for bit."""
    x, target = (v.cuda() for v in data(70, 64, dtype))

    def build():
        model = Stack(dtype=dtype).cuda()
        return model, G.FusedAdamW(model.parameters(), lr=1e-2, state_bits=bits, max_grad_norm=1.0, seed=3)

    def step_of(model, opt):
        def step():
            opt.zero_grad(set_to_none=False)
            loss = loss_of(*model(x), target)
            loss.backward()
            return loss.detach()

        return step

    a, oa = build()
    step = step_of(a, oa)
    for _ in range(8):
        step()
        oa.step()
    b, ob = build()
    graphed = GraphedStep(step_of(b, ob), warmup=3, optimizer=ob)
    for _ in range(5):
        graphed()
        torch.cuda.synchronize()
    for (name, p), q in zip(a.named_parameters(), b.parameters()):
        assert torch.isfinite(p.float()).all() and torch.equal(p, q), name
    assert float(oa.grad_norm) == float(ob.grad_norm)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_single_rows_of_a_batch(dtype):
    """Rows one by one, as in generating, against the same rows in a batch that takes other kernels.  Sums of up to 160 terms in another order:
    184 half steps of fp32 of their absolute sum in each of two blocks, times what the norms stretch them by, and a step of the type wherever
    a rounding falls on the other side; 16 of those steps of the largest value in all."""
    model = Stack(dtype=dtype).cuda().eval()
    x, _ = data(48, 64, dtype)
    x = x.cuda()
    with torch.no_grad():
        s, h = model(x)
        for i in (0, 7, 47):
            s1, h1 = model(x[i:i + 1])
            for one, all_ in ((s1, s), (h1, h)):
                step = max(torch.finfo(dtype).eps, 184 * EPS32)
                assert (one[0].float() - all_[i].float()).abs().max() <= 16 * step * all_.float().abs().max()
