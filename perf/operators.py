"""The measured cases of the residual-block operators: a Linear with its epilogue (`gcpnet_amd.linear_act`), the norms around a block
with its gate and residual scale (`gcpnet_amd.residual_norm`), and the AdamW step over many tensors (`gcpnet_amd.FusedAdamW`).

`run` computes a case in plain torch operations, or, where `own` is true, through this package's calls; `exact` evaluates the
definitions in float64."""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BLOCK = 256  # elements that share a scale of the 8-bit optimizer states
E4M3_MIN_NORMAL, E4M3_STEP = 2.0 ** -6, 2.0 ** -9


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one step of generating for four sequences: a wide layer, all of it the read of the weights
        dict(name="linear_four_rows_bf16", op="linear", rows=4, k=4096, n=8192, type="bf16", act="silu", bias=True, residual=False, train=False),
        # the readout head of a batch of 16 graphs, 100 -> 200 as in the LBA model: latency is all there is
        dict(name="linear_readout_fp32", op="linear", rows=16, k=100, n=200, type="fp32", act="silu", bias=True, residual=False, train=True),
        # a feed-forward layer on the node rows of the 10 000-node graph, 128 -> 512
        dict(name="linear_nodes_fp32", op="linear", rows=10000, k=128, n=512, type="fp32", act="silu", bias=True, residual=False, train=True),
        # odd sizes, as vocabularies and trimmed batches have them
        dict(name="linear_odd_fp16", op="linear", rows=1537, k=1000, n=777, type="fp16", act="leakyrelu", bias=True, residual=True, train=True),
        # the closing layer of a block in training, its residual stream added in the epilogue
        dict(name="linear_train_bf16", op="linear", rows=8192, k=4096, n=4096, type="bf16", act="silu", bias=True, residual=True, train=True),
        # one generated token between two blocks
        dict(name="norm_one_row_bf16", op="norm", rows=1, d=4096, type="bf16", gate="channel", gate_act=None, post="rms", pre="rms", train=False),
        # node rows of the 10 000-node graph at its width of 128, layer norms with biases
        dict(name="norm_nodes_fp32", op="norm", rows=10000, d=128, type="fp32", gate="channel", gate_act=None, post="layer", pre="layer", train=True),
        # the residual stream of a large model in training, with a gate of its own for every element
        dict(name="norm_train_bf16", op="norm", rows=16384, d=4096, type="bf16", gate="element", gate_act="sigmoid", post="rms", pre="rms", train=True),
        # the tensors of one GCPInteractions layer and a norm limit: many small ones
        dict(name="adamw_layer_fp32", op="adamw", tensors=90, elements=300000, type="fp32", bits=32, clip=True),
        # a model of 100 million parameters, states in fp32
        dict(name="adamw_100m_fp32", op="adamw", tensors=24, elements=100000000, type="fp32", bits=32, clip=False),
        # the same with bf16 parameters and states in 8 bits
        dict(name="adamw_100m_bf16_8bit", op="adamw", tensors=24, elements=100000000, type="bf16", bits=8, clip=False),
        # a middling model in fp32 with states in 8 bits and a norm limit
        dict(name="adamw_5m_fp32_8bit", op="adamw", tensors=40, elements=5000000, type="fp32", bits=8, clip=True),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(("linear", "norm", "adamw"))
    kind = rng.choice(("fp32", "bf16", "fp16"))
    if op == "linear":
        train = rng.random() < 0.6
        rows = _spread(rng, 1, 16384) if train else _spread(rng, 1, 512)
        k, n = _spread(rng, 16, 6000), _spread(rng, 16, 6000)
        if rng.random() < 0.6:  # most layers are multiples of 8 wide
            k, n = -(-k // 8) * 8, -(-n // 8) * 8
        most = (8192 * 4096 * 4096) // (1 if kind != "fp32" else 8)
        if rows * k * n > most:
            rows = max(1, most // (k * n))
        acts = (None, "silu", "sigmoid") if kind == "fp32" else (None, "relu", "leakyrelu", "selu", "silu", "sigmoid")
        return dict(op=op, rows=rows, k=k, n=n, type=kind, act=rng.choice(acts), bias=rng.random() < 0.7, residual=rng.random() < 0.5, train=train)
    if op == "norm":
        d = _spread(rng, 16, 8192)
        if rng.random() < 0.6:
            d = -(-d // 8) * 8
        rows = min(_spread(rng, 1, 60000), (16384 * 4096) // (d * (2 if kind == "fp32" else 1)))
        gate = rng.choice((None, "channel", "element"))
        return dict(op=op, rows=rows, d=d, type=kind, gate=gate, gate_act=rng.choice((None, "sigmoid", "silu")) if gate else None,
                    post=rng.choice((None, "layer", "rms")), pre=rng.choice(("layer", "rms")), train=rng.random() < 0.7)
    return dict(op=op, tensors=_spread(rng, 1, 120), elements=_spread(rng, 3000, 60000000), type=rng.choice(("fp32", "bf16")), bits=rng.choice((8, 32)),
                clip=rng.random() < 0.5)


def work(case):
    t = 4 if case["type"] == "fp32" else 2
    if case["op"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        one = m * k + n * k + m * n + n * case["bias"]
        b = one + m * n * case["residual"]
        if not case["train"]:
            return {"bytes": t * b, "flops": 2 * m * n * k}
        # forward, then dy in and dx, dw, db out (the gradient of the residual is dy itself)
        return {"bytes": t * (b + m * n + m * k + n * k + n * case["bias"]), "flops": 6 * m * n * k}
    if case["op"] == "norm":
        rd = case["rows"] * case["d"]
        gate = {None: 0, "channel": case["d"], "element": rd}[case["gate"]]
        small = case["d"] * sum({None: 0, "rms": 1, "layer": 2}[case[w]] for w in ("post", "pre"))
        b = 4 * rd + gate + small
        return {"bytes": t * (2 * b if case["train"] else b), "flops": (60 if case["train"] else 20) * rd}
    n = sum(_sizes(case))
    master = 0 if case["type"] == "fp32" else 8
    states = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
    return {"bytes": n * (3 * t + master + states), "flops": 20 * n}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _sizes(case):
    """Tensor sizes of an optimizer case: weights and vectors of unequal size, most of the elements in a few."""
    n = case["tensors"]
    share = [1.0 / (1 + (i * 7) % n) for i in range(n)]
    return [max(1, int(case["elements"] * s / sum(share))) for s in share]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    t = DTYPES[case["type"]]

    def normal(*shape, std=1.0, mean=0.0):
        return torch.randn(*shape, generator=g, device="cuda").mul_(std).add_(mean)

    st = dict(case=dict(case))
    if case["op"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        st["x"] = normal(m, k).to(t)
        st["w"] = normal(n, k, std=k ** -0.5).to(t)
        st["b"] = normal(n, std=0.3).to(t) if case["bias"] else None
        st["r"] = normal(m, n, std=2.0).to(t) if case["residual"] else None
        st["dy"] = normal(m, n).to(t) if case["train"] else None
        leaves = ("x", "w", "b", "r")
    elif case["op"] == "norm":
        m, d = case["rows"], case["d"]
        loud = 1.0 + 9.0 * (torch.rand(d, generator=g, device="cuda") < 0.01)  # a residual stream has a few loud channels
        st["x"] = (normal(m, d) * loud).to(t)
        level = torch.exp(normal(m, 1, std=0.5))
        if m > 8:  # padding rows, which a block's mask leaves empty
            level[-(m // 16 + 1):] = 0.0
        st["y"] = (normal(m, d) * level + 0.1 * level).to(t)
        st["gate"] = None if case["gate"] is None else normal(d, std=0.3, mean=0.5).to(t) if case["gate"] == "channel" else normal(m, d).to(t)
        st["scale"] = 0.7
        for w in ("post", "pre"):
            st[w + "_w"] = normal(d, std=0.2, mean=1.0).to(t) if case[w] else None
            st[w + "_b"] = normal(d, std=0.2).to(t) if case[w] == "layer" else None
        st["ds"], st["dh"] = (normal(m, d).to(t), normal(m, d).to(t)) if case["train"] else (None, None)
        leaves = ("x", "y", "gate", "post_w", "post_b", "pre_w", "pre_b")
    else:
        return _prepare_adamw(case, g, t, st)
    if case["train"]:
        for name in leaves:
            if st[name] is not None:
                st[name].requires_grad_()
    return st


def _prepare_adamw(case, g, t, st):
    """Parameters, gradients and moments of a run that is under way.  The tensors are views of flat buffers in which each begins at
    a multiple of 256 elements, the rest of its last 256 being zero."""
    sizes = _sizes(case)
    blocks = [-(-s // BLOCK) for s in sizes]
    nb = sum(blocks)
    dev = "cuda"
    per = torch.tensor(blocks, device=dev)
    first = torch.cumsum(per, 0) - per
    tensor = torch.repeat_interleave(torch.arange(len(sizes), device=dev), per)
    size = torch.tensor(sizes, device=dev)
    at = (torch.arange(nb, device=dev) - first[tensor])[:, None] * BLOCK + torch.arange(BLOCK, device=dev)
    inside = at < size[tensor][:, None]
    level = torch.exp(torch.randn(nb, 1, generator=g, device=dev) * 1.5 - 7.0)  # gradients differ in size from layer to layer
    zero = torch.rand(nb, 1, generator=g, device=dev) < 0.03                    # rows that a batch did not reach
    noise = lambda: torch.randn(nb, BLOCK, generator=g, device=dev)  # noqa: E731
    master = noise().mul_(0.02).mul_(inside)
    grad = noise().mul_(level).mul_(inside & ~zero)
    m = (noise() * level).mul_(0.3).mul_(inside)
    v = (noise().square_().mul_(0.3).add_(0.7) * level.square()).mul_(inside)
    st.update(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, seed=17, max_norm=1.0 if case["clip"] else None,
              param=master.to(t), grad=grad.to(t), master=None, step=torch.full((), 12.0, device=dev), at=at, tensor=tensor)
    if t != torch.float32:
        st["master"] = master
    if case["bits"] == 32:
        st.update(m=m, v=v, m_scale=None, v_scale=None)
    else:
        st["m_scale"], st["v_scale"] = _block_scale(m), _block_scale(v)
        st["m"] = (m / st["m_scale"]).to(torch.float8_e4m3fn)
        st["v"] = (v / st["v_scale"]).clamp_(min=E4M3_STEP).mul_(v > 0).to(torch.float8_e4m3fn)
    if own:
        import gcpnet_amd

        def views(flat, width=BLOCK):
            starts = (first * width).tolist()
            return [flat.view(-1)[a:a + (s if width == BLOCK else b)] for a, s, b in zip(starts, sizes, blocks)]

        params = [torch.nn.Parameter(p) for p in views(st["param"])]
        for p, gr in zip(params, views(st["grad"])):
            p.grad = gr
        opt = gcpnet_amd.FusedAdamW(params, lr=st["lr"], betas=st["betas"], eps=st["eps"], weight_decay=st["weight_decay"],
                                    state_bits=case["bits"], max_grad_norm=st["max_norm"], seed=st["seed"])
        names = dict(exp_avg=("m", BLOCK), exp_avg_sq=("v", BLOCK), exp_avg_scale=("m_scale", 1), exp_avg_sq_scale=("v_scale", 1), master=("master", BLOCK))
        parts = {k: views(st[f], w) for k, (f, w) in names.items() if st[f] is not None}
        for i, p in enumerate(params):
            opt.state[p].update({k: part[i] for k, part in parts.items()}, step=st["step"].clone())
        st["opt"] = opt
    return st


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(st):
    return {"linear": _run_linear, "norm": _run_norm, "adamw": _run_adamw}[st["case"]["op"]](st)


def _act(kind, z):
    if kind == "relu":
        return torch.where(z > 0, z, 0.0)
    if kind == "leakyrelu":
        return torch.where(z > 0, z, 0.01 * z)
    if kind == "selu":
        return 1.0507009873554805 * torch.where(z > 0, z, 1.6732632423543772 * (torch.exp(torch.where(z > 0, 0.0, z)) - 1))
    if kind == "silu":
        return z / (1 + torch.exp(-z))
    if kind == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    return z


def _act_slope(kind, z):
    if kind == "relu":
        return torch.where(z > 0, 1.0, 0.0)
    if kind == "leakyrelu":
        return torch.where(z > 0, 1.0, 0.01)
    if kind == "selu":
        return 1.0507009873554805 * torch.where(z > 0, 1.0, 1.6732632423543772 * torch.exp(torch.where(z > 0, 0.0, z)))
    s = 1 / (1 + torch.exp(-z))
    if kind == "silu":
        return s * (1 + z * (1 - s))
    return s * (1 - s)


def _run_linear(st):
    c = st["case"]
    x, w, b, r, dy = (st[k] for k in ("x", "w", "b", "r", "dy"))
    if own:
        import gcpnet_amd

        if not c["train"]:
            with torch.no_grad():
                return {"y": gcpnet_amd.linear_act(x, w, b, act=c["act"], residual=r)}
        y = gcpnet_amd.linear_act(x, w, b, act=c["act"], residual=r)
        named = [(k, st[k]) for k in ("x", "w", "b", "r") if st[k] is not None]
        grads = torch.autograd.grad(y, [v for _, v in named], dy)
        return {"y": y.detach(), **{"d" + k: g for (k, _), g in zip(named, grads)}}
    with torch.no_grad():
        t = x.dtype
        xf, wf = x.float(), w.float()
        z = torch.matmul(xf, wf.t())
        if b is not None:
            z = z + b.float()
        y = _act(c["act"], z)
        if r is not None:
            y = y + r.float()
        out = {"y": y.to(t)}
        if c["train"]:
            g = dy.float()
            dz = g if c["act"] is None else g * _act_slope(c["act"], z)
            out["dx"] = torch.matmul(dz, wf).to(t)
            out["dw"] = torch.matmul(dz.t(), xf).to(t)
            if b is not None:
                out["db"] = dz.sum(0).to(t)
            if r is not None:
                out["dr"] = dy
        return out


def _norm_stats(kind, a, eps):
    mean = a.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(a[:, :1])
    c = a - mean
    rstd = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + eps)
    return c * rstd, rstd


def _norm_back(kind, n, rstd, dn):
    out = dn - n * (dn * n).mean(1, keepdim=True)
    if kind == "layer":
        out = out - dn.mean(1, keepdim=True)
    return out * rstd


def _norm_plain(st, wide):
    """The operator and its gradients in the type `wide`; every result in that type."""
    c, eps = st["case"], 1e-5
    f = lambda k: None if st[k] is None else st[k].detach().to(wide)  # noqa: E731
    x, y, gate = f("x"), f("y"), f("gate")
    wp, bp, wq, bq = f("post_w"), f("post_b"), f("pre_w"), f("pre_b")
    u, n1, r1 = y, None, None
    if c["post"]:
        n1, r1 = _norm_stats(c["post"], y, eps)
        u = n1 * wp if bp is None else n1 * wp + bp
    a = None if gate is None else _act(c["gate_act"], gate)
    s = x + st["scale"] * (u if a is None else u * a)
    n2, r2 = _norm_stats(c["pre"], s, eps)
    h = n2 * wq if bq is None else n2 * wq + bq
    out = {"s": s, "h": h}
    if c["train"]:
        ds, dh = f("ds"), f("dh")
        out["dpre_w"] = (dh * n2).sum(0)
        if bq is not None:
            out["dpre_b"] = dh.sum(0)
        gs = ds + _norm_back(c["pre"], n2, r2, dh * wq)
        out["dx"] = gs
        du = st["scale"] * (gs if a is None else gs * a)
        if a is not None:
            dg = st["scale"] * gs * u
            if c["gate_act"]:
                dg = dg * _act_slope(c["gate_act"], gate)
            out["dgate"] = dg if c["gate"] == "element" else dg.sum(0)
        if c["post"]:
            out["dpost_w"] = (du * n1).sum(0)
            if bp is not None:
                out["dpost_b"] = du.sum(0)
            du = _norm_back(c["post"], n1, r1, du * wp)
        out["dy"] = du
    return out


def _run_norm(st):
    c = st["case"]
    if not own:
        with torch.no_grad():
            return {k: v.to(st["x"].dtype) for k, v in _norm_plain(st, torch.float32).items()}
    import gcpnet_amd

    call = lambda: gcpnet_amd.residual_norm(  # noqa: E731
        st["x"], st["y"], st["gate"], scale=st["scale"], gate_act=c["gate_act"], post=c["post"], post_weight=st["post_w"], post_bias=st["post_b"],
        pre=c["pre"], pre_weight=st["pre_w"], pre_bias=st["pre_b"], eps=1e-5)
    if not c["train"]:
        with torch.no_grad():
            s, h = call()
        return {"s": s, "h": h}
    s, h = call()
    named = [(k, st[k]) for k in ("x", "y", "gate", "post_w", "post_b", "pre_w", "pre_b") if st[k] is not None]
    grads = torch.autograd.grad((s, h), [v for _, v in named], (st["ds"], st["dh"]))
    return {"s": s.detach(), "h": h.detach(), **{"d" + k: g for (k, _), g in zip(named, grads)}}


def _block_scale(a):
    """The power of two that takes a block's largest finite magnitude into (224, 448], the end of e4m3's range."""
    top = torch.where(torch.isfinite(a), a.abs(), 0.0).amax(1, keepdim=True)
    e = ((top.view(torch.int32) + 0x1FFFFF) >> 23) - 8
    return (e.clamp(min=1) << 23).view(torch.float32)


def _mix(h):
    """A bijection of 32-bit values (in int64): two multiply-xorshift rounds."""
    h = h ^ (h >> 16)
    h = (h * 0x7FEB352D) & 0xFFFFFFFF
    h = h ^ (h >> 15)
    h = (h * 0x846CA68B) & 0xFFFFFFFF
    return h ^ (h >> 16)


def _random_bits(st):
    """20 bits for each element, from (seed, number of the tensor, step, number of the element)."""
    k = _mix((st["seed"] + 0x9E3779B9 * st["tensor"]) & 0xFFFFFFFF)
    k = _mix(k ^ st["step"].to(torch.int64))
    return _mix((k[:, None] + st["at"]) & 0xFFFFFFFF) & 0xFFFFF


def _e4m3_stochastic(y, bits):
    """y in [0, 448] to a value of e4m3, up with the probability of its place between two; never to 0 from above 0."""
    whole = ((y.view(torch.int32) + bits.to(torch.int32)) & -0x100000).view(torch.float32)
    small = torch.floor(y * 512.0 + bits.to(torch.float32) * 2.0 ** -20) * E4M3_STEP
    small = torch.where((y > 0) & (small == 0), E4M3_STEP, small)
    return torch.where(y >= E4M3_MIN_NORMAL, whole, small)


def _run_adamw(st):
    if own:
        st["opt"].step()
        out = {"grad_norm": st["opt"].grad_norm}
    else:
        with torch.no_grad():
            out = _adamw_plain(st)
    out.update(param=st["param"], master=st["master"], exp_avg=st["m"], exp_avg_sq=st["v"], exp_avg_scale=st["m_scale"], exp_avg_sq_scale=st["v_scale"])
    return {k: v for k, v in out.items() if v is not None}


def _adamw_plain(st):
    b1, b2 = st["betas"]
    g = st["grad"].float()
    norm = None
    if st["max_norm"] is not None:
        norm = torch.sqrt((g * g).sum())
        g = g * torch.clamp(st["max_norm"] / (norm + 1e-6), max=1.0)
    st["step"] += 1
    t = st["step"].double()
    lr1 = (st["lr"] / (1 - b1 ** t)).float()
    root2 = torch.sqrt(1 - b2 ** t).float()
    eight = st["m_scale"] is not None
    m, v = (st["m"].float() * st["m_scale"], st["v"].float() * st["v_scale"]) if eight else (st["m"], st["v"])
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * (1 - b2)) * g
    p = st["param"] if st["master"] is None else torch.where(st["master"].to(st["param"].dtype) == st["param"], st["master"], st["param"].float())
    p = p * (1 - st["lr"] * st["weight_decay"]) - lr1 * (m / (torch.sqrt(v) / root2 + st["eps"]))
    st["param"].copy_(p)
    if st["master"] is not None:
        st["master"].copy_(p)
    if eight:
        st["m_scale"], st["v_scale"] = _block_scale(m), _block_scale(v)
        code = torch.where(torch.isfinite(m), m * (1 / st["m_scale"]), math.nan)
        st["m"].copy_(code)
        code = torch.where(torch.isfinite(v), v * (1 / st["v_scale"]), math.nan)
        st["v"].copy_(torch.where(torch.isnan(code), code, _e4m3_stochastic(code, _random_bits(st))))
    else:
        st["m"].copy_(m)
        st["v"].copy_(v)
    return {"grad_norm": norm}


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return {"linear": _exact_linear, "norm": _exact_norm, "adamw": _exact_adamw}[case["op"]](st)


def _exact_linear(st):
    c = st["case"]
    x, w, b, r, dy = (None if st[k] is None else st[k].detach().double() for k in ("x", "w", "b", "r", "dy"))
    z = x @ w.t()
    if b is not None:
        z += b
    f = {None: lambda a: a, "relu": lambda a: a.clamp(min=0), "leakyrelu": lambda a: torch.maximum(a, 0.01 * a),
         "selu": lambda a: 1.0507009873554805 * (a.clamp(min=0) + 1.6732632423543772 * torch.expm1(a.clamp(max=0))),
         "silu": lambda a: a * torch.sigmoid(a), "sigmoid": torch.sigmoid}[c["act"]]
    out = {"y": f(z) + (0 if r is None else r)}
    if c["train"]:
        with torch.enable_grad():
            leaf = z.detach().requires_grad_()
            (dz,) = torch.autograd.grad(f(leaf) * 1.0, leaf, dy)
        out.update(dx=dz @ w, dw=dz.t() @ x)
        if b is not None:
            out["db"] = dz.sum(0)
        if r is not None:
            out["dr"] = dy
    return out


def _exact_norm(st):
    """By automatic differentiation of the definition."""
    c = st["case"]
    names = ("x", "y", "gate", "post_w", "post_b", "pre_w", "pre_b")
    q = {k: None if st[k] is None else st[k].detach().double().requires_grad_(c["train"]) for k in names}

    def norm(kind, a, w, b):
        if kind is None:
            return a
        if kind == "layer":
            a = a - a.mean(-1, keepdim=True)
        a = a / (a.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * w
        return a if b is None else a + b

    with torch.enable_grad():
        u = norm(c["post"], q["y"], q["post_w"], q["post_b"])
        if q["gate"] is not None:
            u = u * {None: lambda a: a, "sigmoid": torch.sigmoid, "silu": lambda a: a * torch.sigmoid(a)}[c["gate_act"]](q["gate"])
        s = q["x"] + st["scale"] * u
        h = norm(c["pre"], s, q["pre_w"], q["pre_b"])
        out = {"s": s.detach(), "h": h.detach()}
        if c["train"]:
            live = [k for k in names if q[k] is not None]
            grads = torch.autograd.grad((s, h), [q[k] for k in live], (st["ds"].double(), st["dh"].double()))
            out.update({"d" + k: g for k, g in zip(live, grads)})
    return out


def _exact_adamw(st):
    """The codes of 8-bit states have no value here: they are what 32 bits round to, at random."""
    b1, b2 = st["betas"]
    t = float(st["step"]) + 1
    g = st["grad"].double()
    out = {}
    if st["max_norm"] is not None:
        out["grad_norm"] = g.norm()
        g = g * min(1.0, st["max_norm"] / (float(out["grad_norm"]) + 1e-6))
    eight = st["m_scale"] is not None
    m, v = st["m"].double(), st["v"].double()
    if eight:
        m, v = m * st["m_scale"].double(), v * st["v_scale"].double()
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g.square()
    p = (st["param"] if st["master"] is None else st["master"]).double()
    p = p - st["lr"] * st["weight_decay"] * p - st["lr"] * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + st["eps"])
    out["param"] = p
    if st["master"] is not None:
        out["master"] = p
    if not eight:
        out.update(exp_avg=m, exp_avg_sq=v)
    return out
