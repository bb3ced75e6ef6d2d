"""residual_norm (gcpnet_block_norm_forward / _backward) against its formulas in 64 bits on the CPU, forward and all gradients."""
import math

import pytest
import torch

import gcpnet_amd as G
from gcpnet_amd import _lib

EPS32 = 2.0 ** -24
# Half steps of fp32 that a value in the middle may be off, relative to the absolute sum it comes from: a row's sum is formed in at most
# 16 sequential and 10 + 16 tree or wave additions (42), and a handful of products, a root and a quotient follow.
K = 48


def half(t):
    return torch.finfo(t).eps / 2


def act64(kind, g):
    s = 1 / (1 + torch.exp(-g))
    a = {None: g, "sigmoid": s, "silu": g * s, "relu": g.clamp(min=0), "leakyrelu": torch.where(g > 0, g, 0.01 * g)}[kind]
    da = {None: torch.ones_like(g), "sigmoid": s * (1 - s), "silu": s * (1 + g * (1 - s)), "relu": (g > 0).double(),
          "leakyrelu": torch.where(g > 0, 1.0, 0.01).double()}[kind]
    # exp(-g) is off by about |g| + 2 half steps, relatively, the quotient and the products add a few; the derivatives multiply 1 + |g|
    rough = EPS32 * (g.abs() + 8)
    return a, da, rough * a.abs(), rough * ((g.abs() + 8) * da.abs().clamp(max=2) + s * (1 + g.abs()))


def norm64(kind, z, eps):
    if kind is None:
        return z, torch.zeros_like(z[:, :1]), torch.ones_like(z[:, :1])
    mean = z.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(z[:, :1])
    r = 1 / ((z - mean).square().mean(1, keepdim=True) + eps).sqrt()
    return (z - mean) * r, mean, r


def reference(cfg, t, x, y, gate, pw, pb, qw, qb, ds, dh, scale, eps):
    """{name: (value, tolerance)} in float64; `t`: the type of the rows."""
    post, pre, gact = cfg
    D = lambda v: None if v is None else v.detach().cpu().double()  # noqa: E731
    x, y, gate, pw, pb, qw, qb, ds, dh = map(D, (x, y, gate, pw, pb, qw, qb, ds, dh))
    out = {}
    e = K * EPS32
    one = torch.ones_like(x[0])
    n1, mean1, r1 = norm64(post, y, eps)
    w1, b1 = (one if pw is None else pw), (0 * one if pb is None else pb)
    u = n1 * w1 + b1
    d_n1 = e * (y.abs() + mean1.abs()) * r1 if post else 0 * y
    d_u = w1.abs() * d_n1 + e * ((n1 * w1).abs() + b1.abs()) if post else 0 * y
    a, da, d_a, d_da = (one, 0 * one, 0 * one, 0 * one) if gate is None else act64(gact, gate)
    s = x + scale * a * u
    d_s = abs(scale) * (a.abs() * d_u + u.abs() * d_a) + 4 * EPS32 * (x.abs() + (scale * a * u).abs())
    out["s"] = s, d_s + half(t) * (s.abs() + d_s)
    if pre:
        n2, mean2, r2 = norm64(pre, s, eps)
        # an error of the row moves its mean and its root by no more than the mean and the root mean square of the errors
        move = d_s + d_s.mean(1, keepdim=True) + n2.abs() * d_s.square().mean(1, keepdim=True).sqrt()
        w2, b2 = (one if qw is None else qw), (0 * one if qb is None else qb)
        d_n2 = r2 * move + e * (s.abs() + mean2.abs()) * r2
        h = n2 * w2 + b2
        d_h = w2.abs() * d_n2 + 4 * EPS32 * ((n2 * w2).abs() + b2.abs())
        out["h"] = h, d_h + half(t) * (h.abs() + d_h)
    if ds is None:
        return out
    rows = x.shape[0]
    chain = (K + rows / 512) * EPS32

    def column(name, v, tol, kind):
        tot = v.sum(0)
        tol = tol.sum(0) + chain * v.abs().sum(0)
        out[name] = tot, tol + half(kind) * (tot.abs() + tol)

    gs, d_gs = ds, 0 * ds
    if pre:
        dn = dh * w2
        m0, m1 = (dn.mean(1, keepdim=True) if pre == "layer" else 0), (dn * n2).mean(1, keepdim=True)
        d_m1 = (dn.abs() * d_n2).mean(1, keepdim=True) + e * (dn * n2).abs().mean(1, keepdim=True)
        d_m0 = e * dn.abs().mean(1, keepdim=True) if pre == "layer" else 0
        gs = ds + r2 * (dn - m0 - n2 * m1)
        # (r2 moves with the row's error too: relatively as much as the root mean square of the errors times r2)
        rel = r2 * d_s.square().mean(1, keepdim=True).sqrt() + e
        d_gs = r2 * (d_m0 + n2.abs() * d_m1 + d_n2 * m1.abs()) + (rel + e) * r2 * (dn.abs() + abs(m0) + (n2 * m1).abs()) + 4 * EPS32 * ds.abs()
        if qw is not None:
            column("dpre_w", dh * n2, dh.abs() * d_n2, reference.w)
        if qb is not None:
            column("dpre_b", dh, 0 * dh, reference.w)
    out["dx"] = gs, d_gs + half(t) * (gs.abs() + d_gs)
    q, d_q = scale * gs, abs(scale) * d_gs + 2 * EPS32 * (scale * gs).abs()
    du, d_du = a * q, a.abs() * d_q + q.abs() * d_a + EPS32 * (a * q).abs()
    if gate is not None:
        dg = q * u * da
        d_dg = da.abs() * (u.abs() * d_q + q.abs() * d_u) + (q * u).abs() * d_da + 4 * EPS32 * dg.abs()
        if gate.dim() == 1:
            column("dgate", dg, d_dg, t)
        else:
            out["dgate"] = dg, d_dg + half(t) * (dg.abs() + d_dg)
    if post:
        if pw is not None:
            column("dpost_w", du * n1, du.abs() * d_n1 + n1.abs() * d_du, reference.w)
        if pb is not None:
            column("dpost_b", du, d_du, reference.w)
        v, d_v = du * w1, w1.abs() * d_du + EPS32 * (du * w1).abs()
        m0, m1 = (v.mean(1, keepdim=True) if post == "layer" else 0 * v[:, :1]), (v * n1).mean(1, keepdim=True)
        d_m0 = d_v.mean(1, keepdim=True) + e * v.abs().mean(1, keepdim=True)
        d_m1 = (n1.abs() * d_v + v.abs() * d_n1).mean(1, keepdim=True) + e * (v * n1).abs().mean(1, keepdim=True)
        du = r1 * (v - m0 - n1 * m1)
        d_du = r1 * (d_v + d_m0 + n1.abs() * d_m1 + m1.abs() * d_n1) + 2 * e * r1 * (v.abs() + m0.abs() + (n1 * m1).abs())
    out["dy"] = du, d_du + half(t) * (du.abs() + d_du)
    return out


def make(rows, d, t, gate, post, pre, affine, wt=None, seed=0, spread=False):
    g = torch.Generator().manual_seed(seed + 7 * d + rows)
    wt = wt or t
    n = lambda *s, std=1.0, mean=0.0: torch.randn(*s, generator=g) * std + mean  # noqa: E731
    x, y = n(rows, d, std=2.0), n(rows, d) + 0.5
    if rows > 2:
        y[-1] = 0.0  # a row that a mask left empty
        x[-2], y[-2] = 0.0, 0.0
    ten = dict(x=x, y=y, gate={None: None, "channel": n(d), "element": n(rows, d)}[gate])
    for k, kind in (("post", post), ("pre", pre)):
        ten[k + "_weight"] = n(d, std=0.3, mean=1.0) if kind and affine > 0 else None
        ten[k + "_bias"] = n(d, std=0.3) if kind and affine > 1 else None
    out = {}
    for k, v in ten.items():
        if v is None:
            out[k] = None
            continue
        v = v.to(wt if k[:3] in ("pos", "pre") else t).cuda()
        if spread and v.dim() == 2:  # rows inside wider rows
            wide = torch.full((rows, d + 24), 7.0, dtype=v.dtype, device="cuda")
            wide[:, 8:8 + d] = v
            v = wide[:, 8:8 + d]
        out[k] = v.requires_grad_()
    return out, n(rows, d).to(t).cuda(), n(rows, d).to(t).cuda()


def compare(out, want, what=""):
    for k, (v, tol) in want.items():
        got = out[k].detach().cpu().double()
        assert got.shape == v.shape, (k, got.shape)
        # (below the smallest normal number the steps stay as they are: half of one is smallest_normal * eps / 2, 2^-25 for fp16)
        kind = torch.finfo(out[k].dtype)
        tol = tol + kind.smallest_normal * kind.eps / 2
        bad = (got - v).abs() > tol
        # (a value from max + half a step on rounds to infinity: a gradient of a row of zeros, 1 / sqrt(eps) = 316 twice, in fp16)
        bad &= ~(torch.isinf(got) & (got.sign() == v.sign()) & (v.abs() + tol >= kind.max))
        assert not bad.any(), f"{what} {k}: {int(bad.sum())} of {v.numel()} off, worst {float(((got - v).abs() / tol.clamp(min=1e-300)).max()):.3g} of the tolerance"


def both_ways(rows, d, t, gate, gact, post, pre, affine, wt=None, scale=0.7, eps=1e-5, spread=False):
    ten, ds, dh = make(rows, d, t, gate, post, pre, affine, wt, spread=spread)
    reference.w = wt or t
    s, h = G.residual_norm(**ten, scale=scale, gate_act=gact, post=post, pre=pre, eps=eps)
    names = [k for k, v in ten.items() if v is not None]
    outs, gos = ((s, h), (ds, dh)) if h is not None else ((s,), (ds,))
    grads = torch.autograd.grad(outs, [ten[k] for k in names], gos)
    out = dict(s=s, h=h, **{"d" + k.replace("_weight", "_w").replace("_bias", "_b"): g for k, g in zip(names, grads)})
    for k, g in zip(names, grads):
        assert g.dtype == ten[k].dtype and g.shape == ten[k].shape
    want = reference((post, pre, gact), t, ten["x"], ten["y"], ten["gate"], ten["post_weight"], ten["post_bias"], ten["pre_weight"],
                     ten["pre_bias"], ds, dh if pre else None, scale, eps)
    compare(out, want, f"{rows}x{d}")
    return out


SHAPES = [(1, 1), (5, 2), (3, 7), (33, 16), (600, 20), (70, 64), (37, 100), (1100, 128), (9, 257), (4, 512), (6, 513), (3, 1000), (2, 1021),
          (5, 2048), (3, 4096), (2, 4099), (2, 8192), (2, 16384), (1, 16383)]


@pytest.mark.gpu
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,d", SHAPES)
def test_sizes(rows, d, t):
    both_ways(rows, d, t, "channel", "sigmoid", "rms", "layer", 2)
    both_ways(rows, d, t, "element", None, "layer", "rms", 1)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("pre", [None, "layer", "rms"])
@pytest.mark.parametrize("post", [None, "layer", "rms"])
@pytest.mark.parametrize("gate,gact", [(None, None), ("channel", None), ("channel", "silu"), ("element", "sigmoid"), ("element", "leakyrelu")])
def test_forms(gate, gact, post, pre, t):
    both_ways(41, 96, t, gate, gact, post, pre, 0)
    both_ways(41, 96, t, gate, gact, post, pre, 2, wt=torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("wt", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("rows,d", [(9000, 40), (2100, 1000), (1100, 2044), (1100, 4096), (600, 6000), (300, 16000)])
def test_many_rows(rows, d, wt):
    """Several rows a group, with the parameters in LDS or, where there is no room, from memory in every turn."""
    both_ways(rows, d, torch.bfloat16, "channel", "silu", "layer", "layer", 2, wt=wt)
    both_ways(rows, d, torch.bfloat16, "element", "sigmoid", "rms", "rms", 1, wt=wt)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_strided_rows_and_leading_dimensions(t):
    both_ways(50, 128, t, "element", "sigmoid", "rms", "rms", 1, spread=True)
    both_ways(50, 130, t, "element", "sigmoid", "rms", "rms", 1, spread=True)
    g = torch.Generator().manual_seed(0)
    x, y = torch.randn(3, 4, 5, 32, generator=g).to(t).cuda(), torch.randn(4, 3, 5, 32, generator=g).to(t).cuda().transpose(0, 1)
    gate = torch.randn(3, 4, 1, 32, generator=g).to(t).cuda().expand(3, 4, 5, 32)
    s, h = G.residual_norm(x, y, gate, pre="layer")
    s2, h2 = G.residual_norm(x.reshape(60, 32), y.reshape(60, 32), gate.reshape(60, 32), pre="layer")
    assert s.shape == x.shape and torch.equal(s.view(60, 32), s2) and torch.equal(h.view(60, 32), h2)
    one = G.residual_norm(x[0, 0, 0], y[0, 0, 0], pre="rms")  # a row without leading dimensions
    assert one[0].shape == (32,)
    row = torch.randn(32, generator=g).to(t).cuda().expand(60, 32).requires_grad_()  # the same row 60 times, and as a gate
    s, _ = G.residual_norm(row, y.reshape(60, 32), row, pre="rms")
    (dr,) = torch.autograd.grad(s, row, torch.ones_like(s))
    want = 1 + y.reshape(60, 32).double()
    assert ((dr.double() - want).abs() <= 2 * half(t) * (1 + want.abs())).all()
    transposed = torch.randn(32, 60, generator=g).to(t).cuda().t()
    assert torch.equal(G.residual_norm(transposed, pre="rms")[1], G.residual_norm(transposed.contiguous(), pre="rms")[1])


@pytest.mark.gpu
@pytest.mark.parametrize("off", [1, 4, 8])
def test_addresses_off_16_bytes(off):
    """Rows, parameters and gradients that begin anywhere."""
    g = torch.Generator().manual_seed(off)
    d, rows = 64, 9
    flat = lambda n: torch.randn(n + off, generator=g).bfloat16().cuda()[off:]  # noqa: E731
    ten = dict(x=flat(rows * d).view(rows, d), y=flat(rows * d).view(rows, d), gate=flat(d), post_weight=flat(d), post_bias=flat(d),
               pre_weight=flat(d), pre_bias=flat(d))
    ten = {k: v.requires_grad_() for k, v in ten.items()}
    ds, dh = flat(rows * d).view(rows, d), flat(rows * d).view(rows, d)
    reference.w = torch.bfloat16
    s, h = G.residual_norm(**ten, post="layer", pre="rms")
    grads = torch.autograd.grad((s, h), list(ten.values()), (ds, dh))
    names = ("dx", "dy", "dgate", "dpost_w", "dpost_b", "dpre_w", "dpre_b")
    want = reference(("layer", "rms", None), torch.bfloat16, *ten.values(), ds, dh, 1.0, 1e-5)
    compare(dict(s=s, h=h, **dict(zip(names, grads))), want)


@pytest.mark.gpu
def test_a_norm_alone_and_gradients_of_one_output():
    x = (torch.randn(20, 48, generator=torch.Generator().manual_seed(0)) * 3 + 1).cuda().requires_grad_()
    w = torch.linspace(0.5, 1.5, 48).cuda().requires_grad_()
    s, h = G.residual_norm(x, pre="layer", pre_weight=w)
    assert s is x
    want = torch.nn.functional.layer_norm(x.double(), (48,), w.double())
    up = torch.randn(20, 48, generator=torch.Generator().manual_seed(1)).cuda()
    g1 = torch.autograd.grad(h, (x, w), up)
    g2 = torch.autograd.grad(want, (x, w), up.double())
    for a, b in zip(g1, g2):  # (sums of 48 or 20 terms of at most 5, roots of at least 1/3)
        assert (a - b).abs().max() < K * EPS32 * 50
    y = torch.randn(20, 48, generator=torch.Generator().manual_seed(2)).cuda().requires_grad_()
    s, h = G.residual_norm(x, y, scale=0.5, pre="rms")
    assert torch.equal(torch.autograd.grad(s, y, up, retain_graph=True)[0], up * 0.5)
    only_h = torch.autograd.grad(h, (x, y), up, retain_graph=True)
    both = torch.autograd.grad((s, h), (x, y), (torch.zeros_like(up), up))
    assert torch.equal(only_h[0], both[0]) and torch.equal(only_h[1], both[1])


@pytest.mark.gpu
def test_gradients_against_differences():
    g = torch.Generator().manual_seed(4)
    ten = dict(x=torch.randn(3, 12, generator=g), y=torch.randn(3, 12, generator=g), gate=torch.randn(12, generator=g),
               post_weight=torch.randn(12, generator=g), pre_weight=torch.randn(12, generator=g))
    up = torch.randn(2, 3, 12, generator=g)
    leaf = {k: v.clone().cuda().requires_grad_() for k, v in ten.items()}
    kw = dict(gate_act="silu", post="rms", pre="layer", eps=1e-3)
    s, h = G.residual_norm(**leaf, **kw)
    grads = torch.autograd.grad((s, h), list(leaf.values()), (up[0].cuda(), up[1].cuda()))
    for (k, v), got in zip(ten.items(), grads):
        way = torch.randn(v.shape, generator=g)
        step = 2.0 ** -7

        def at(f):
            p = {q: (w + f * step * way if q == k else w).cuda() for q, w in ten.items()}
            s, h = G.residual_norm(**p, **kw)
            return float((s.double().cpu() * up[0]).sum() + (h.double().cpu() * up[1]).sum())

        # (four-point differences: the fifth derivative times step^4 = 4e-9 against values of order 10 to 100, and 1e-5 / step of rounding)
        slope = (8 * (at(1) - at(-1)) - (at(2) - at(-2))) / (12 * step)
        want = float((got.cpu().double() * way).sum())
        assert abs(slope - want) < 2e-2 * max(1.0, abs(want)), k


@pytest.mark.gpu
def test_no_rows_one_row_and_repeats():
    x = torch.zeros(0, 40, device="cuda", requires_grad=True)
    w = torch.ones(40, device="cuda", requires_grad=True)
    s, h = G.residual_norm(x, torch.zeros(0, 40, device="cuda"), w, pre="rms", pre_weight=w)
    assert s.shape == h.shape == (0, 40)
    (s.sum() + h.sum()).backward()
    assert float(w.grad.abs().sum()) == 0.0 and x.grad.shape == (0, 40)
    a = both_ways(2000, 128, torch.bfloat16, "channel", "sigmoid", "rms", "layer", 2)
    b = both_ways(2000, 128, torch.bfloat16, "channel", "sigmoid", "rms", "layer", 2)
    for k in a:
        assert torch.equal(a[k], b[k]), k


@pytest.mark.gpu
def test_saved_tensors_that_went_to_the_host_and_second_derivatives():
    ten, ds, dh = make(20, 64, torch.float32, "element", "rms", "layer", 2)
    names = list(ten)
    call = lambda: G.residual_norm(**ten, gate_act="silu", post="rms", pre="layer")  # noqa: E731
    want = torch.autograd.grad(call(), [ten[k] for k in names], (ds, dh))
    with torch.autograd.graph.save_on_cpu():
        out = call()
    for p, q in zip(torch.autograd.grad(out, [ten[k] for k in names], (ds, dh)), want):
        assert torch.equal(p, q)
    got = torch.autograd.grad(call(), [ten[k] for k in names], (ds, dh), create_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    with pytest.raises(RuntimeError):
        got[0].sum().backward()


@pytest.mark.gpu
def test_infinities_stay_in_their_rows():
    x, y = torch.randn(6, 32, device="cuda"), torch.randn(6, 32, device="cuda")
    y[2, 3], x[4, 0] = math.inf, math.nan
    s, h = G.residual_norm(x, y, post="layer", pre="rms")
    for out in (s, h):
        assert torch.isfinite(out[[0, 1, 3, 5]]).all() and not torch.isfinite(out[[2, 4]]).all(1).any()


@pytest.mark.gpu
def test_captured_and_on_another_stream():
    g = torch.Generator().manual_seed(0)
    x, y = (torch.randn(300, 256, generator=g).cuda().bfloat16() for _ in range(2))
    w = torch.rand(256, generator=g).cuda().bfloat16().requires_grad_()
    x.requires_grad_()
    up = torch.randn(300, 256, generator=g).cuda().bfloat16()

    def step():
        s, h = G.residual_norm(x, y, w, post="rms", pre="rms", pre_weight=w)
        return (s.detach(), h.detach(), *torch.autograd.grad((s, h), (x, w), (up, up)))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(3):
        with torch.no_grad():
            x.add_(0.25)
            y.mul_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, step())), k


def test_refusals():
    x = torch.zeros(2, 8)
    with pytest.raises(_lib.GcpnetHipError, match="GPU"):
        G.residual_norm(x, pre="rms")
    with pytest.raises(TypeError):
        G.residual_norm([1.0], pre="rms")
    lib = _lib.load()
    n = _lib.BlockNorm()
    n.rows, n.d, n.type, n.param_type, n.x, n.x_ld, n.eps = 4, 8, 0, 0, 4096, 8, 1e-5
    call = lambda: lib.gcpnet_block_norm_forward(n, None, 4096, None, None)  # noqa: E731
    for field, bad, code in (("d", 0, -1), ("rows", -1, -1), ("type", 3, -1), ("param_type", 1, -1), ("pre", 3, -1), ("post", 1, -1), ("gate", 4096, -1),
                             ("act", 9, -1), ("x_ld", -8, -1), ("d", 16385, -2), ("rows", 1 << 33, -2), ("x", None, -1)):
        keep = getattr(n, field)
        setattr(n, field, bad)
        assert call() == code, field
        setattr(n, field, keep)
    n.pre = 1
    assert lib.gcpnet_block_norm_forward(n, None, None, None, None) == -1  # (pre without h)
    assert lib.gcpnet_block_norm_backward(n, None, *[None] * 11) == -1  # (pre without statistics)
    n.rows = 0
    assert call() == 0
    n.rows = -1
    assert lib.gcpnet_block_norm_backward_scratch(n) == -1


def test_more_threads_than_a_launch_takes():
    n = _lib.BlockNorm()
    n.rows, n.d, n.x, n.x_ld, n.eps, n.pre = 1 << 30, 8, 4096, 8, 1e-5, 1
    assert _lib.load().gcpnet_block_norm_forward(n, None, 4096, None, None) == -2


@pytest.mark.gpu
@pytest.mark.parametrize("act", [None, "relu", "leakyrelu", "selu", "silu", "sigmoid"])
def test_a_gate_that_is_nan_stays_in_its_row(act):
    x, y, gate = (torch.randn(6, 32, device="cuda") for _ in range(3))
    gate[2, 3] = math.nan
    s, h = G.residual_norm(x, y, gate, gate_act=act, pre="rms")
    assert torch.isnan(s[2, 3]) and torch.isnan(h[2]).all() and int(torch.isnan(s).sum()) == 1 and torch.isfinite(h[[0, 1, 3, 4, 5]]).all()


@pytest.mark.gpu
def test_refusals_of_tensors():
    x, w = torch.zeros(2, 8, device="cuda"), torch.ones(8, device="cuda")
    for kw in (dict(pre="batch"), dict(pre=None), dict(post="rms"), dict(gate=w), dict(y=torch.zeros(2, 4, device="cuda")), dict(eps=-1.0),
               dict(y=x, gate=torch.zeros(2, 1, device="cuda")), dict(pre="rms", pre_weight=torch.ones(4, device="cuda")),
               dict(y=x, post_weight=w), dict(y=x, gate=w, gate_act="gate")):
        with pytest.raises(ValueError):
            G.residual_norm(x, **kw)
    for kw in (dict(y=x.half()), dict(pre_weight=w.half()), dict(pre_weight=w.double()), dict(pre_weight=2.0)):
        with pytest.raises(TypeError):
            G.residual_norm(x, **kw)
    with pytest.raises(TypeError):
        G.residual_norm(x.bfloat16(), pre_weight=w.bfloat16(), pre_bias=w)
    with pytest.raises(TypeError):
        G.residual_norm(x.double())
    with pytest.raises(_lib.GcpnetHipError):
        G.residual_norm(x, x.cpu())
    with pytest.raises(ValueError):
        G.residual_norm(torch.zeros(1, 16385, device="cuda"))
