"""linear_act where values leave the range or the resolution of their type: pre-activations beyond the largest number of the rows' type, and
SELU close to 0."""
import pytest
import torch

import gcpnet_amd as G
from tests.test_linear_act import EPS32, both_ways, half, make

LA, AL = 1.0507009873554805, 1.6732632423543772
# act'(z) far below and far above 0
SLOPES = {None: (1.0, 1.0), "relu": (0.0, 1.0), "leakyrelu": (0.01, 1.0), "selu": (0.0, LA), "silu": (0.0, 1.0), "sigmoid": (0.0, 0.0)}


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [5, 40])
@pytest.mark.parametrize("act", list(SLOPES))
@pytest.mark.parametrize("t", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_slopes_beyond_the_range_of_the_type(t, act, rows):
    """One z that is finite in fp32 and beyond the largest number of the rows' type; dy is 1 there and 0 elsewhere, so each gradient has one
    row or element.  dz = act' rounds once (half a step, and the fp32 values before it some 4 EPS32), its product with an operand once more."""
    i, j = 3, 2
    g = torch.Generator().manual_seed(rows)
    for side in (0, 1):
        x, w = torch.randn(rows, 24, generator=g).to(t), (torch.randn(16, 24, generator=g) / 8).to(t)
        sign = 2 * side - 1
        if t == torch.float16:  # +-70000
            x[i], w[j] = 0, 0
            x[i, 0], w[j, 0] = 280, sign * 250
        else:  # +-(2 - 2^-9) 2^127: the largest bf16 number is (2 - 2^-7) 2^127
            x[i], w[j] = 0, 0
            x[i, :2] = 2.0 ** 64
            w[j, 0], w[j, 1] = sign * (2 - 2 ** -7) * 2.0 ** 63, sign * 0.75 * 2 ** -7 * 2.0 ** 63
        z = (x[i].double() * w[j].double()).sum()
        assert torch.finfo(t).max < abs(z) < torch.finfo(torch.float32).max and torch.isinf(z.to(t))
        dy = torch.zeros(rows, 16, dtype=t)
        dy[i, j] = 1
        gx, gw = x.cuda().requires_grad_(), w.cuda().requires_grad_()
        b = torch.zeros(16, device="cuda", requires_grad=True)
        y = G.linear_act(gx, gw, b, act=act)
        if side == 0 and act in ("relu", "selu", "silu", "sigmoid"):
            assert torch.isfinite(y).all()
        dx, dw, db = torch.autograd.grad(y, (gx, gw, b), dy.cuda())
        slope = SLOPES[act][side]
        want = dict(dx=torch.zeros(rows, 24).double(), dw=torch.zeros(16, 24).double(), db=torch.zeros(16).double())
        want["dx"][i], want["dw"][j], want["db"][j] = slope * w[j].double(), slope * x[i].double(), slope
        for name, got in dict(dx=dx, dw=dw, db=db).items():
            off = (got.cpu().double() - want[name]).abs()
            assert (off <= (2.1 * half(t) + 4 * EPS32) * want[name].abs()).all(), (side, name, got[i if name == "dx" else j])


@pytest.mark.gpu
@pytest.mark.parametrize("act", [None, "relu", "leakyrelu", "selu", "silu", "sigmoid"])
@pytest.mark.parametrize("rows,k,n", [(9, 24, 40), (150, 72, 136)])
def test_a_large_negative_value_among_others(rows, k, n, act):
    """fp16: one z of about -70000 in a row and a column of ordinary ones; finite outputs and all gradients as the formulas have them."""
    x, w, b, r, dy = make(rows, k, n, torch.float16)
    with torch.no_grad():
        x[3, 5], w[7, 5] = 280.0, -250.0
        if act is None:  # (y itself would be infinite)
            x[3, 5] = 200.0
    out = both_ways(x, w, b, act, r, dy)
    assert all(torch.isfinite(v).all() for v in out.values())


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [5, 40])
def test_selu_close_to_zero(rows):
    """selu(z) = la al (exp(z) - 1) below 0, to its relative precision however small z is: exp(z) - 1 to 2 units (4 half steps), the
    constant 1, products 2, the bias-free sum of one product 1."""
    z = -torch.logspace(-8, 1, 4 * rows).reshape(rows, 4)
    z[0, 0] = -1e-30
    eye = torch.eye(4, device="cuda")
    y = G.linear_act(z.cuda(), eye, act="selu").cpu().double()
    want = LA * AL * torch.expm1(z.double())
    assert ((y - want).abs() <= 8 * EPS32 * want.abs()).all(), float(((y - want) / want).abs().max())
    gate = z.reshape(-1).cuda()
    s, _ = G.residual_norm(torch.zeros(3, 4 * rows, device="cuda"), torch.ones(3, 4 * rows, device="cuda"), gate, gate_act="selu", pre="rms")
    want = want.reshape(-1)
    assert ((s[1].cpu().double() - want).abs() <= 8 * EPS32 * want.abs()).all()
