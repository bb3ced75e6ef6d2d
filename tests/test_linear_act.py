"""linear_act (gcpnet_linear_act_forward / _backward) against the formulas in 64 bits, forward and all gradients."""
import math

import pytest
import torch

import gcpnet_amd as G
from gcpnet_amd import _lib

EPS32 = 2.0 ** -24
T = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def half(t):
    return torch.finfo(t).eps / 2


def rounded(v, tol, t):
    """The tolerance of a value stored in type t that was `tol` off before: half a step, of a subnormal number below the normal ones."""
    return tol + half(t) * (v.abs() + tol) + torch.finfo(t).smallest_normal * half(t)


def act64(kind, z):
    """act(z), act'(z), and by how much the fp32 evaluations of both may be off (exp(-z): about |z| + 2 half steps, relatively)."""
    s = 1 / (1 + torch.exp(-z))
    e = torch.exp(z.clamp(max=0))
    la, al = 1.0507009873554805, 1.6732632423543772
    a, da = {None: lambda: (z, torch.ones_like(z)), "relu": lambda: (z.clamp(min=0), (z > 0).double()),
             "leakyrelu": lambda: (torch.where(z > 0, z, 0.01 * z), torch.where(z > 0, 1.0, 0.01).double()),
             "selu": lambda: (la * torch.where(z > 0, z, al * (e - 1)), la * torch.where(z > 0, torch.ones_like(z), al * e)),
             "silu": lambda: (z * s, s * (1 + z * (1 - s))), "sigmoid": lambda: (s, s * (1 - s))}[kind]()
    rough = EPS32 * (z.abs() + 8)
    return a, da, rough * (a.abs() + (2 if kind == "selu" else 0)), rough * ((z.abs() + 8) * (da.abs() + s) if kind in ("silu", "sigmoid") else 2 * da.abs())


def second(kind, z):
    """A bound of |act''|, by which an error of z enters act'."""
    return {None: 0.0, "silu": 0.5, "sigmoid": 0.1, "selu": 1.76, "relu": 0.0, "leakyrelu": 0.0}[kind] + 0 * z


def sums(k):
    """Half steps of fp32 that a sum of k products may be off, relative to the sum of their magnitudes: the matrix instructions add k in
    order (at most k), split sums add a few; the products of 16-bit factors are exact, those of fp32 round once."""
    return (k + 24) * EPS32


def reference(x, w, b, act, r, dy, t, bt):
    """{name: (value, tolerance)}.  Where z is nearer to 0 than its error, act' of a kinked activation may be either side's."""
    D = lambda v: None if v is None else v.detach().cpu().double()  # noqa: E731
    x, w, b, r, dy = map(D, (x, w, b, r, dy))
    rows, k = x.shape
    n = w.shape[0]
    z = x @ w.t() + (0 if b is None else b)
    d_z = sums(k) * (x.abs() @ w.abs().t()) + 2 * EPS32 * ((0 if b is None else b.abs()) + z.abs())
    a, da, d_a, d_da = act64(act, z)
    top = torch.maximum(da.abs(), torch.tensor(1.76 if act == "selu" else 1.1))  # (act is Lipschitz with it)
    y = a + (0 if r is None else r)
    d_y = top * d_z + d_a + 2 * EPS32 * (a.abs() + (0 if r is None else r.abs()))
    out = {"y": (y, rounded(y, d_y, t))}
    if dy is None:
        return out
    d_zs = rounded(z, d_z, t) if act is not None else 0 * z  # (stored in the rows' type)
    d_da = d_da + second(act, z) * d_zs
    if act in ("relu", "leakyrelu", "selu"):
        jump = {"relu": 1.0, "leakyrelu": 0.99, "selu": 0.71}[act]
        d_da = d_da + jump * (z.abs() <= d_zs).double()
    dz = dy * da
    d_dz = dy.abs() * d_da + EPS32 * dz.abs()
    db, d_db = dz.sum(0), d_dz.sum(0) + sums(rows) * dz.abs().sum(0)
    d_op = rounded(dz, d_dz, t) if act is not None else 0 * dz  # (an operand in the rows' type; without an activation dy itself)
    dx = dz @ w
    out["dx"] = dx, rounded(dx, d_op @ w.abs() + sums(n) * (dz.abs() @ w.abs()), t)
    dw = dz.t() @ x
    out["dw"] = dw, rounded(dw, d_op.t() @ x.abs() + sums(rows) * (dz.abs().t() @ x.abs()), t)
    if b is not None:
        out["db"] = db, rounded(db, d_db, bt)
    if r is not None:
        out["dr"] = dy, 0 * dy
    return out


def compare(out, want, what=""):
    for name, (v, tol) in want.items():
        got = out[name].detach().cpu().double()
        assert got.shape == v.shape, (name, got.shape, v.shape)
        off = (got - v).abs()
        bad = ~(off <= tol)
        assert not bad.any(), f"{what} {name}: {int(bad.sum())} of {v.numel()} off, worst {float((off / tol.clamp(min=1e-300)).max()):.3g} of the tolerance"


def make(rows, k, n, t, bias=True, residual=True, bt=None, seed=0):
    g = torch.Generator().manual_seed(seed + rows + 3 * k + 7 * n)
    f = lambda *s, std=1.0: torch.randn(*s, generator=g) * std  # noqa: E731
    x, w = f(rows, k).to(t).cuda(), f(n, k, std=k ** -0.5).to(t).cuda()
    b = f(n).to(bt or t).cuda() if bias else None
    return x, w, b, f(rows, n).to(t).cuda() if residual else None, f(rows, n).to(t).cuda()


def both_ways(x, w, b, act, r, dy, what=""):
    leaves = {key: v.requires_grad_() for key, v in dict(dx=x, dw=w, db=b, dr=r).items() if v is not None}
    y = G.linear_act(x, w, b, act=act, residual=r)
    out = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)), y=y)
    for key, v in leaves.items():
        assert out[key].dtype == v.dtype and out[key].shape == v.shape
    want = reference(x, w, b, act, r, dy, x.dtype, x.dtype if b is None else b.dtype)
    compare(out, want, what)
    return out


SHAPES = [(1, 1, 1), (1, 64, 64), (2, 3, 5), (3, 100, 200), (4, 512, 768), (7, 33, 130), (16, 100, 200), (16, 1031, 48), (17, 257, 31), (32, 2048, 40), (33, 64, 65), (64, 128, 64), (64, 1500, 33),
          (65, 136, 72), (130, 200, 20), (129, 96, 257), (300, 64, 512), (515, 72, 136), (1000, 20, 24), (257, 1030, 264), (64, 2056, 128), (2000, 40, 56)]


@pytest.mark.gpu
@pytest.mark.parametrize("t", list(T))
@pytest.mark.parametrize("rows,k,n", SHAPES)
def test_sizes(rows, k, n, t):
    x, w, b, r, dy = make(rows, k, n, T[t])
    both_ways(x, w, b, "silu", r, dy, what=f"{rows}x{k}x{n}")


@pytest.mark.gpu
@pytest.mark.parametrize("t", list(T))
@pytest.mark.parametrize("act", [None, "relu", "leakyrelu", "selu", "silu", "sigmoid"])
def test_forms(act, t):
    for bias, residual in ((True, True), (False, True), (True, False), (False, False)):
        x, w, b, r, dy = make(70, 48, 88, T[t], bias, residual, bt=torch.float32 if residual else None)
        both_ways(x, w, b, act, r, dy)


@pytest.mark.gpu
@pytest.mark.parametrize("t", list(T))
@pytest.mark.parametrize("rows,k,n", [(2304, 320, 2048), (4096, 512, 1096), (700, 3000, 650)])
def test_large(rows, k, n, t):
    """Sizes of each tile of the kernel, more than one band of tiles, ends inside tiles on every side."""
    x, w, b, r, dy = make(rows, k, n, T[t])
    both_ways(x, w, b, "silu", r, dy)


@pytest.mark.gpu
@pytest.mark.parametrize("t", list(T))
def test_strides_and_addresses(t):
    """Rows inside wider rows, operands off 16 bytes, leading dimensions, transposed operands, a broadcast residual."""
    t = T[t]
    x, w, b, r, dy = make(90, 64, 96, t)
    want = both_ways(x, w, b, "silu", r, dy)

    def inside(v, lead, more):
        wide = torch.full((v.shape[0], v.shape[1] + more), 9.0, dtype=t, device="cuda")
        wide[:, lead:lead + v.shape[1]] = v.detach()
        return wide[:, lead:lead + v.shape[1]]

    for lead, more in ((8, 24), (0, 8), (1, 5), (4, 12)):
        got = both_ways(inside(x, lead, more), inside(w, lead, more), b, "silu", inside(r, lead, more), inside(dy, lead, more))
        for key in want:  # (the order of the products' sums does not go by the layout; that of the column sums does)
            assert key == "db" or torch.equal(got[key], want[key]), (lead, key)
    got = both_ways(x.detach().t().contiguous().t(), w.detach().t().contiguous().t(), b, "silu", r, dy.t().contiguous().t())
    for key in want:
        assert torch.equal(got[key], want[key]), key
    y = G.linear_act(x.detach().view(3, 5, 6, 64), w, b, act="silu", residual=r.view(3, 5, 6, 96))
    assert y.shape == (3, 5, 6, 96) and torch.equal(y.reshape(90, 96), want["y"])
    assert torch.equal(G.linear_act(x[4], w, b, act="silu", residual=r[4]), G.linear_act(x[4:5], w, b, act="silu", residual=r[4:5])[0])
    row = r.detach()[:1].clone().requires_grad_()
    y = G.linear_act(x.detach(), w.detach(), b.detach(), residual=row.expand(90, 96))
    (dr,) = torch.autograd.grad(y, row, dy)
    s = dy.double().sum(0, keepdim=True)
    # (torch adds the 90 rows, in fp32 or in steps of the type)
    assert ((dr.double() - s).abs() <= 90 * (EPS32 if t == torch.float32 else half(t)) * dy.double().abs().sum(0)).all()


@pytest.mark.gpu
def test_some_gradients_only_and_no_rows():
    x, w, b, r, dy = make(30, 24, 40, torch.bfloat16)
    want = both_ways(x, w, b, "silu", r, dy)
    for key, leaf in dict(dx=x, dw=w, db=b, dr=r).items():
        others = [v.detach() for v in (x, w, b, r)]
        at = ("dx", "dw", "db", "dr").index(key)
        others[at] = leaf
        y = G.linear_act(others[0], others[1], others[2], act="silu", residual=others[3])
        assert torch.equal(torch.autograd.grad(y, leaf, dy)[0], want[key]), key
    for act in (None, "silu"):
        e = torch.zeros(0, 24, device="cuda", requires_grad=True)
        w2, b2 = torch.ones(40, 24, device="cuda", requires_grad=True), torch.ones(40, device="cuda", requires_grad=True)
        y = G.linear_act(e, w2, b2, act=act)
        assert y.shape == (0, 40)
        y.sum().backward()
        assert e.grad.shape == (0, 24) and float(w2.grad.abs().sum()) == 0.0 and float(b2.grad.abs().sum()) == 0.0


@pytest.mark.gpu
@pytest.mark.parametrize("t", list(T))
def test_infinities_and_large_numbers_stay_in_their_rows(t):
    x, w, b, r, _ = make(40, 72, 48, T[t])
    clean = G.linear_act(x, w, b, residual=r)
    x[3, 5], x[17, 71] = math.inf, math.nan
    y = G.linear_act(x, w, b, residual=r)
    rest = [i for i in range(40) if i not in (3, 17)]
    assert torch.equal(y[rest], clean[rest]) and not torch.isfinite(y[[3, 17]]).any()
    if t != "fp16":
        big = torch.full((5, 40), 1e30, device="cuda", dtype=T[t])
        tiny = torch.full((9, 40), 1e-30, device="cuda", dtype=T[t])
        y = G.linear_act(big, tiny).double()
        want = float(big[0, 0]) * float(tiny[0, 0]) * 40
        assert ((y - want).abs() <= (half(T[t]) + sums(40)) * want).all()


@pytest.mark.gpu
def test_gradients_against_differences():
    x, w, b, r, dy = make(6, 9, 7, torch.float32)
    got = both_ways(x, w, b, "silu", r, dy)
    g = torch.Generator().manual_seed(0)
    ten = dict(dx=x.detach().cpu(), dw=w.detach().cpu(), db=b.detach().cpu(), dr=r.detach().cpu())
    for key, v in ten.items():
        way, step = torch.randn(v.shape, generator=g), 2.0 ** -7

        def at(f):
            p = [(u + f * step * way if q == key else u).cuda() for q, u in ten.items()]
            return float((G.linear_act(p[0], p[1], p[2], act="silu", residual=p[3]).double() * dy.double()).sum())

        # (four-point differences: the fifth derivative times step^4 = 4e-9, and 1e-5 / step of rounding)
        slope = (8 * (at(1) - at(-1)) - (at(2) - at(-2))) / (12 * step)
        want = float((got[key].cpu().double() * way).sum())
        assert abs(slope - want) < 1e-2 * max(1.0, abs(want)), key


@pytest.mark.gpu
def test_saved_tensors_that_went_to_the_host_and_second_derivatives():
    x, w, b, r, dy = make(50, 64, 72, torch.bfloat16)
    leaves = [v.requires_grad_() for v in (x, w, b)]
    want = torch.autograd.grad(G.linear_act(x, w, b, act="silu", residual=r), leaves, dy)
    with torch.autograd.graph.save_on_cpu():
        y = G.linear_act(x, w, b, act="silu", residual=r)
    torch.empty(1 << 20, device="cuda").fill_(math.nan)
    for p, q in zip(torch.autograd.grad(y, leaves, dy), want):
        assert torch.equal(p, q)
    got = torch.autograd.grad(G.linear_act(x, w, b, act="silu", residual=r), leaves, dy, create_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    with pytest.raises(RuntimeError):
        got[0].sum().backward()


@pytest.mark.gpu
def test_repeats_captured_and_on_another_stream():
    """A split product (few tiles, long k) and a large one, bit for bit from run to run, on another stream, and in replays of a graph."""
    for rows, k, n in ((40, 4096, 72), (700, 256, 520)):
        x, w, b, r, dy = make(rows, k, n, torch.bfloat16)
        leaves = [v.requires_grad_() for v in (x, w, b)]

        def step():
            y = G.linear_act(x, w, b, act="silu", residual=r)
            return (y.detach(), *torch.autograd.grad(y, leaves, dy))

        want = step()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = step()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        del got
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        for _ in range(3):
            with torch.no_grad():
                x.mul_(0.75)
                w.add_(0.001)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(held, step()))
        del graph, held


def test_refusals():
    x, w = torch.zeros(2, 8), torch.zeros(4, 8)
    with pytest.raises(_lib.GcpnetHipError, match="GPU"):
        G.linear_act(x, w)
    with pytest.raises(TypeError):
        G.linear_act(1.0, w)
    lib = _lib.load()
    q = _lib.LinearDesc()
    q.rows, q.k, q.n, q.x, q.w, q.x_ld, q.w_ld = 4, 8, 12, 4096, 4096, 8, 8
    call = lambda y=None: lib.gcpnet_linear_act_forward(q, None, 0, y, None, None, None)  # noqa: E731
    assert call() == -1  # (no y)
    for field, bad, code in (("k", 0, -1), ("n", 0, -1), ("rows", -1, -1), ("type", 3, -1), ("bias_type", 2, -1), ("act", 6, -1), ("x", None, -1),
                             ("w", None, -1), ("x_ld", -1, -1), ("rows", 1 << 33, -2), ("k", 1 << 21, -2), ("n", 1 << 21, -2)):
        keep = getattr(q, field)
        setattr(q, field, bad)
        assert call(4096) == code, field
        setattr(q, field, keep)
    q.act = 4
    assert lib.gcpnet_linear_act_backward(q, None, 4096, 12, None, None, None, None, None) == -1  # (no z)
    q.act = 0
    assert lib.gcpnet_linear_act_backward(q, None, 4096, 12, None, None, 4096, None, None) == -1  # (db without workspace)
    assert lib.gcpnet_linear_act_workspace(q, 0) == 0 and lib.gcpnet_linear_act_forward(q, None, 0, 4096, None, 8, None) == -1  # (off 16 bytes)
    q.x = 4098  # (off 16 bytes, a copy of 4 rows of 8 floats; in a backward dz and the column sums of 512 groups too)
    assert lib.gcpnet_linear_act_workspace(q, 0) == 0 and lib.gcpnet_linear_act_workspace(q, 1) == 32 + 48 + 512 * 12
    q.rows = 65  # (a few rows need no copies)
    assert lib.gcpnet_linear_act_workspace(q, 0) == 65 * 8
    q.rows = 4
    q.type = 7
    assert lib.gcpnet_linear_act_workspace(q, 0) == -1
    q.type = 0
    q.rows = 0
    assert call() == 0


def test_more_workgroups_than_a_launch_takes():
    q = _lib.LinearDesc()
    q.rows, q.k, q.n, q.x, q.w, q.x_ld, q.w_ld = 1 << 30, 4, 4, 4096, 4096, 4, 4
    assert _lib.load().gcpnet_linear_act_forward(q, None, 0, 4096, None, 4096, None) == -2


def test_every_tile_is_visited_once():
    """The order of the tiles (a model of gcp_tile_of_block) is a permutation, also where their number is no multiple of 8."""
    for tiles_m in (1, 2, 7, 8, 9, 17, 40):
        for tiles_n in (1, 3, 8, 13):
            total, seen = tiles_m * tiles_n, set()
            for block in range(total):
                xcd, at = block & 7, block >> 3
                i = xcd * (total >> 3) + min(xcd, total & 7) + at
                first = i // (8 * tiles_n) * 8
                high = min(8, tiles_m - first)
                rest = i % (8 * tiles_n)
                seen.add((first + rest % high, rest // high))
            assert seen == {(a, b) for a in range(tiles_m) for b in range(tiles_n)}


@pytest.mark.gpu
def test_refusals_of_tensors():
    x, w = torch.zeros(2, 8, device="cuda"), torch.zeros(4, 8, device="cuda")
    for args, kw in (((x, w.t()), {}), ((x, w[0]), {}), ((x, w, x[0]), {}), ((x, w), dict(act="gate")), ((x, w), dict(residual=x)),
                     ((x, torch.zeros(0, 8, device="cuda")), {}), ((x[:, :0], w[:, :0]), {})):
        with pytest.raises(ValueError):
            G.linear_act(*args, **kw)
    for args in ((x, w.half()), (x.double(), w.double()), (x.half(), w.half(), w[:, 0].bfloat16())):
        with pytest.raises(TypeError):
            G.linear_act(*args)
    with pytest.raises(_lib.GcpnetHipError):
        G.linear_act(x, w.cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("act", [None, "relu", "leakyrelu", "selu", "silu", "sigmoid"])
@pytest.mark.parametrize("rows", [5, 40])
def test_nan_passes_every_activation(rows, act):
    x, w, b, r, _ = make(rows, 72, 48, torch.float32)
    x[3, 5] = math.nan
    y = G.linear_act(x, w, b, act, residual=r)
    assert torch.isnan(y[3]).all() and torch.isfinite(y[[i for i in range(rows) if i != 3]]).all()
