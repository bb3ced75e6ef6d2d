"""FusedAdamW (gcpnet_grad_norm / gcpnet_adamw_begin / gcpnet_adamw_step) against the update in 64 bits, and its 8-bit moments code for
code against an integer model of their rounding on the CPU."""
import copy
import math

import pytest
import torch

import gcpnet_amd as G
from gcpnet_amd import _lib

EPS = 2.0 ** -24  # half a step of fp32, relative
E4M3 = torch.float8_e4m3fn


# ---------------------------------------------------------------------------------------------------------------- the model
def _mix(h):
    h = h ^ (h >> 16)
    h = (h * 0x7FEB352D) & 0xFFFFFFFF
    h = h ^ (h >> 15)
    h = (h * 0x846CA68B) & 0xFFFFFFFF
    return h ^ (h >> 16)


def block_scale(a):
    """[blocks, 256] fp32 -> the power of two that takes the largest finite magnitude into (224, 448], at least 2^-126."""
    top = torch.where(torch.isfinite(a), a.abs(), torch.zeros_like(a)).amax(1)
    mant, e = torch.frexp(top)  # top = mant 2^e, mant in [1/2, 1)
    k = e - 9 + (mant > 0.875).to(e.dtype)
    k = torch.where(top == 0, torch.full_like(k, -126), k).clamp(min=-126)
    return torch.ldexp(torch.ones_like(top), k)


def blocks_of(x):
    pad = -x.numel() % 256
    return torch.nn.functional.pad(x.reshape(-1), (0, pad)).view(-1, 256)


def encode(m, v, step, seed=0, ordinal=0, first=0):
    """fp32 moments (flat, CPU) -> e4m3 codes as bytes and scales.  `first`: the index of element 0 (a multiple of 256)."""
    n = m.numel()
    bm, bv = blocks_of(m), blocks_of(v)
    sm, sv = block_scale(bm), block_scale(bv)
    ym, yv = bm / sm[:, None], bv / sv[:, None]
    i = torch.arange(bm.numel(), dtype=torch.int64).view(bm.shape) + first
    key = _mix(_mix(torch.tensor((seed + 0x9E3779B9 * ordinal) & 0xFFFFFFFF)) ^ step)
    high = i >> 32
    key = torch.where(high > 0, _mix(key ^ _mix(high)), key)
    r = _mix((key + (i & 0xFFFFFFFF)) & 0xFFFFFFFF) & 0xFFFFF
    whole = ((yv.view(torch.int32) + r.to(torch.int32)) & -0x100000).view(torch.float32)
    small = torch.floor((yv.double() * 512 + r.double() * 2.0 ** -20).float()) / 512
    small = torch.where((yv > 0) & (small == 0), torch.full_like(small, 1 / 512), small)
    cv = torch.where(yv >= 2.0 ** -6, whole, small)
    cm = torch.where(torch.isfinite(bm), ym, torch.full_like(ym, math.nan)).to(E4M3).view(torch.uint8)
    cv = torch.where(torch.isfinite(bv), cv, torch.full_like(cv, math.nan)).to(E4M3).view(torch.uint8)
    return cm.view(-1)[:n], cv.view(-1)[:n], sm, sv


def decode(codes, scale):
    n = codes.numel()
    return (blocks_of(codes.view(E4M3).float()) * scale[:, None]).view(-1)[:n]


def update64(p, g, m, v, t, lr, b1, b2, eps, wd, clip=1.0):
    p, g, m, v = (a.double() for a in (p, g, m, v))
    g = g * clip
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    u = lr / (1 - b1 ** t) * m / (v.sqrt() / math.sqrt(1 - b2 ** t) + eps)
    return p * (1 - lr * wd) - u, m, v, u


def check_update(got_p, got_m, got_v, p, g, m, v, t, lr, b1, b2, eps, wd, clip=1.0):
    """One step against 64 bits.  m: the factors, two products and a sum round, 4 half steps of |b1 m| + |(1 - b1) g| (6 with the
    clipped gradient); v: the same with g twice, 8; p: two roundings of p (keep, product) and one of the difference, and the update's
    own: m 6, v / 2 4, the root (a unit in the last place) 2, its correction and their product 2, the sum with eps 1, the reciprocal (a
    unit) 2, its product 1, lr's correction and the product 2 -- 20 -- and 4 for products of these, where b1 m and (1 - b1) g do not
    cancel, which enters as their absolute sum."""
    wp, wm, wv, u = update64(p, g, m, v, t, lr, b1, b2, eps, wd, clip)
    mass = (b1 * m.double()).abs() + ((1 - b1) * g.double() * clip).abs()
    assert ((got_m.double() - wm).abs() <= 6 * EPS * mass + 1e-44).all()
    assert ((got_v.double() - wv).abs() <= 8 * EPS * wv + 1e-44).all()
    root = wv.sqrt() / math.sqrt(1 - b2 ** t) + eps
    tol = 3 * EPS * p.double().abs() + 24 * EPS * lr / (1 - b1 ** t) * mass / root + EPS * wp.abs() + 1e-44
    assert ((got_p.double() - wp).abs() <= tol).all(), ((got_p.double() - wp).abs() / tol).max()


def start(n, dtype=torch.float32, seed=0, offset=0):
    g = torch.Generator().manual_seed(seed + n)
    buf = torch.zeros(n + offset, dtype=dtype, device="cuda")
    p = torch.nn.Parameter(buf[offset:])
    p.data.copy_(torch.randn(n, generator=g))
    p.grad = torch.zeros(n + offset, dtype=dtype, device="cuda")[offset:]
    return p, g


def gradient(p, g, level=0.01):
    x = torch.randn(p.shape, generator=g) * level * torch.exp(2 * torch.randn(p.shape, generator=g))
    x[torch.rand(p.shape, generator=g) < 0.1] = 0
    return x.to(p.dtype)


# ---------------------------------------------------------------------------------------------------------------- refusals
def test_refusals():
    w = torch.nn.Parameter(torch.zeros(3))
    for kw in (dict(state_bits=16), dict(lr=-1.0), dict(eps=-1.0), dict(betas=(1.0, 0.9)), dict(weight_decay=-0.1), dict(max_grad_norm=0.0)):
        with pytest.raises(ValueError):
            G.FusedAdamW([w], **kw)
    with pytest.raises(TypeError):
        G.FusedAdamW([w], lr=torch.tensor(1e-3))
    with pytest.raises(TypeError):
        G.FusedAdamW([torch.nn.Parameter(torch.zeros(3, dtype=torch.float16))])
    opt = G.FusedAdamW([w])
    with pytest.raises(TypeError):
        opt.add_param_group(dict(params=[torch.nn.Parameter(torch.zeros(3, dtype=torch.float64))]))
    assert len(opt.param_groups) == 1
    opt.step()  # (no gradient: nothing to do)
    w.grad = torch.ones(3)
    with pytest.raises(_lib.GcpnetHipError, match="GPU"):
        opt.step()


def test_a_parameter_twice_is_refused():
    w = torch.nn.Parameter(torch.zeros(3))
    with pytest.warns(UserWarning), pytest.raises(ValueError, match="twice"):
        G.FusedAdamW([w, w])


def test_bad_arguments_at_the_c_entries():
    lib = _lib.load()
    arr = (_lib.AdamWTensor * 1)()
    arr[0].n = 5  # (pointers all NULL)
    assert lib.gcpnet_grad_norm(1, arr, 0, 16, None) == _lib.E_BADARG
    assert lib.gcpnet_adamw_begin(1, arr, 1e-3, 0.9, 0.999, 16, None, 0, 0.0, None, None) == _lib.E_BADARG
    assert lib.gcpnet_adamw_step(1, arr, 0, 32, 1e-3, 0.9, 0.999, 1e-8, 0.0, 16, None, 0, None) == _lib.E_BADARG
    assert lib.gcpnet_adamw_step(0, None, 2, 32, 1e-3, 0.9, 0.999, 1e-8, 0.0, None, None, 0, None) == _lib.E_BADARG
    assert lib.gcpnet_adamw_step(0, None, 0, 16, 1e-3, 0.9, 0.999, 1e-8, 0.0, None, None, 0, None) == _lib.E_BADARG
    arr[0].n = -1
    assert lib.gcpnet_grad_norm_partials(1, arr) == _lib.E_BADARG
    arr[0].n = 16385
    assert lib.gcpnet_grad_norm_partials(1, arr) == 2


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_state_dict_keeps_the_types_of_the_state(bits, dtype):
    def state(p):
        kind = torch.float32 if bits == 32 else E4M3
        st = dict(step=torch.tensor(3.0), exp_avg=torch.randn(5, 70).to(kind), exp_avg_sq=torch.rand(5, 70).to(kind))
        if bits == 8:
            st.update(exp_avg_scale=torch.rand(2), exp_avg_sq_scale=torch.rand(2))
        if dtype == torch.bfloat16:
            st["master"] = torch.randn(5, 70)
        return st

    a = torch.nn.Parameter(torch.randn(5, 70).to(dtype))
    o1 = G.FusedAdamW([a], state_bits=bits, seed=5)
    o1.state[a] = state(a)
    b = torch.nn.Parameter(torch.zeros(5, 70, dtype=dtype))
    o2 = G.FusedAdamW([b], state_bits=bits)
    o2.load_state_dict(copy.deepcopy(o1.state_dict()))
    assert o2.param_groups[0]["seed"] == 5
    for k, v in o1.state[a].items():
        w = o2.state[b][k]
        assert w.dtype == v.dtype and w is not v and torch.equal(w.float(), v.float()), k
    o3 = G.FusedAdamW([b], state_bits=40 - bits)  # moments of the other kind
    d = o1.state_dict()
    d["param_groups"][0]["state_bits"] = 40 - bits
    with pytest.raises(_lib.GcpnetHipError):
        o3.load_state_dict(d)


def test_the_model_of_the_codes():
    """The rounding model used below: scales, exact values, expectation of the stochastic rounding."""
    x = torch.tensor([0.0, 1.0, 1.75, 1.7500002, 2.0, 1e-45, 3e38])
    s = block_scale(torch.nn.functional.pad(x[:, None], (0, 255)))
    y = x.double() / s.double()
    assert (y <= 448).all() and (y[1:5] > 224).all() and y[6] > 224 and s[0] == 2.0 ** -126
    v = torch.full((256 * 4096,), 0.3)
    v[::256] = 1.0
    _, cv, _, sv = encode(v, v, 1)
    d = decode(cv, sv)
    assert torch.equal(d[::256], v[::256])
    d = d.view(-1, 256)[:, 1:]
    # 0.3 lies between two codes an eighth of its power of two (1/4) apart: sd <= 1/64, the mean of 10^6 within 6 sd / 1000
    assert abs(float(d.double().mean()) - 0.3) < 6 / 64 / 1000
    assert set(d.unique().tolist()) == {0.28125, 0.3125}


# ---------------------------------------------------------------------------------------------------------------- updates
SIZES = [1, 3, 255, 256, 257, 4095, 4096, 4097, 70001]


@pytest.mark.gpu
@pytest.mark.parametrize("clip", [None, 0.5])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_steps_against_64_bits(dtype, bits, clip):
    """Four steps of tensors of all lengths, some at odd addresses; every step is checked from the state before it."""
    lr, b1, b2, eps, wd, seed = 3e-3, 0.9, 0.99, 1e-8, 0.05, 1234
    ps = [start(n, dtype, offset=k % 3) for k, n in enumerate(SIZES)]
    opt = G.FusedAdamW([p for p, _ in ps], lr=lr, betas=(b1, b2), eps=eps, weight_decay=wd, state_bits=bits, max_grad_norm=clip, seed=seed)
    for t in range(1, 5):
        for p, g in ps:
            p.grad.copy_(gradient(p, g, 0.0 if t == 4 else 0.01))
        before = [{k: v.detach().cpu().clone() for k, v in opt.state[p].items()} for p, _ in ps]
        old = [p.detach().cpu().clone() for p, _ in ps]
        opt.step()
        coef = 1.0
        if clip is not None:
            norm = math.sqrt(sum(float(p.grad.double().square().sum()) for p, _ in ps))
            assert abs(float(opt.grad_norm) - norm) <= 20 * EPS * norm
            coef = min(1.0, clip / (float(opt.grad_norm) + 1e-6))
        for k, (p, _) in enumerate(ps):
            st = {key: v.cpu() for key, v in opt.state[p].items()}
            b = before[k]
            n = p.numel()
            assert float(st["step"]) == t
            zero = torch.zeros(n)
            if bits == 8:
                m0 = decode(b["exp_avg"].view(torch.uint8), b["exp_avg_scale"]) if b else zero
                v0 = decode(b["exp_avg_sq"].view(torch.uint8), b["exp_avg_sq_scale"]) if b else zero
            else:
                m0, v0 = (b["exp_avg"], b["exp_avg_sq"]) if b else (zero, zero)
            p0 = b["master"] if b and dtype == torch.bfloat16 else old[k].float()
            p1 = st["master"] if dtype == torch.bfloat16 else p.detach().cpu()
            g = p.grad.cpu().float()
            f = torch.float32
            m1 = m0 * torch.tensor(b1, dtype=f) + (g * torch.tensor(coef, dtype=f)) * torch.tensor(1 - b1, dtype=f)
            gc = g * torch.tensor(coef, dtype=f)
            v1 = v0 * torch.tensor(b2, dtype=f) + (gc * torch.tensor(1 - b2, dtype=f)) * gc
            if bits == 32:
                m1, v1 = st["exp_avg"], st["exp_avg_sq"]
            check_update(p1, m1, v1, p0, g, m0, v0, t, lr, b1, b2, eps, wd, coef)
            if dtype == torch.bfloat16:
                assert torch.equal(p.detach().cpu(), p1.to(dtype))
            if bits == 8 and clip is None:  # (a clipped gradient may differ from the model's in its last bit)
                cm, cv, sm, sv = encode(m1, v1, t, seed, k)
                assert torch.equal(st["exp_avg_scale"], sm) and torch.equal(st["exp_avg_sq_scale"], sv)
                assert torch.equal(st["exp_avg"].view(torch.uint8), cm) and torch.equal(st["exp_avg_sq"].view(torch.uint8), cv)


@pytest.mark.gpu
def test_many_tensors_and_groups():
    """More tensors than one launch of each kernel takes, in two groups and two types, some without a gradient or without elements."""
    g = torch.Generator().manual_seed(0)
    ps = [torch.nn.Parameter(torch.randn(1 + i % 7, 3, generator=g).cuda()) for i in range(500)]
    qs = [torch.nn.Parameter(torch.randn(i % 5, generator=g).cuda().to(torch.bfloat16)) for i in range(60)]
    for p in ps + qs:
        p.grad = torch.randn(p.shape, generator=g).to(p.dtype).cuda()
    ps[3].grad = None
    ref = [copy.deepcopy(p.detach().cpu()) for p in ps + qs]
    opt = G.FusedAdamW([dict(params=ps, lr=1e-2), dict(params=qs, lr=1e-1, weight_decay=0.0, state_bits=8)], max_grad_norm=3.0)
    opt.step()
    live = [p for p in ps + qs if p.grad is not None]
    norm = math.sqrt(sum(float(p.grad.double().square().sum()) for p in live))
    assert abs(float(opt.grad_norm) - norm) <= 20 * EPS * norm
    assert torch.equal(ps[3].detach().cpu(), ref[3]) and not opt.state[ps[3]]
    for p, r in zip(ps + qs, ref):
        if p.grad is None:
            continue
        half = p.dtype == torch.bfloat16
        z = torch.zeros(p.shape)
        want, _, _, _ = update64(r.float(), p.grad.cpu().float(), z, z, 1, 1e-1 if half else 1e-2, 0.9, 0.999, 1e-8, 0.0 if half else 1e-2, 3.0 / norm)
        got = opt.state[p]["master"] if half else p.detach()
        # (a first step moves every element by lr (1 + 24 half steps), p rounds three times)
        assert ((got.cpu().double() - want).abs() <= 24 * EPS * (r.float().abs().double() + 0.1) + 1e-9).all()


@pytest.mark.gpu
def test_same_as_torch_over_a_run_and_state_dicts_interchange():
    """Ten steps like torch.optim.AdamW's in 64 bits; its fp32 state_dict after five is continued here, and ours there."""
    g = torch.Generator().manual_seed(3)
    shapes = [(33, 17), (5,), (64, 3, 3)]
    init = [torch.randn(s, generator=g) for s in shapes]
    grads = [[torch.randn(s, generator=g) for s in shapes] for _ in range(10)]
    kw = dict(lr=1e-2, betas=(0.8, 0.95), eps=1e-6, weight_decay=0.1)

    def run(ps, make, sequence):
        opt = make(ps)
        for k, gs in enumerate(sequence):
            if k == 5:
                d = copy.deepcopy(opt.state_dict())
                opt = (G.FusedAdamW if type(opt) is torch.optim.AdamW else torch.optim.AdamW)(ps, **kw)
                opt.load_state_dict(d)
            for p, x in zip(ps, gs):
                p.grad = x.to(p)
            opt.step()
        return ps

    want = [torch.nn.Parameter(p.double()) for p in init]
    opt = torch.optim.AdamW(want, **kw)
    for gs in grads:
        for p, x in zip(want, gs):
            p.grad = x.double()
        opt.step()
    for first in (G.FusedAdamW, torch.optim.AdamW):
        got = run([torch.nn.Parameter(p.cuda()) for p in init], lambda ps: first(ps, **kw), grads)
        for a, b in zip(got, want):
            # (ten steps, each within 24 half steps of |p| + the update; |p| <= 5)
            assert (a.detach().cpu().double() - b).abs().max() <= 10 * 24 * EPS * 5


@pytest.mark.gpu
def test_layouts():
    """A permuted parameter, and gradients with other strides than their parameter's; a slice is refused."""
    g = torch.Generator().manual_seed(1)
    x, gr = torch.randn(40, 30, generator=g), torch.randn(40, 30, generator=g)
    plain = torch.nn.Parameter(x.clone().cuda())
    turned = torch.nn.Parameter(x.t().contiguous().cuda().t())
    spread = torch.nn.Parameter(x.clone().cuda())
    plain.grad, turned.grad = gr.cuda(), gr.cuda()
    spread.grad = torch.stack((gr, gr), -1).cuda()[..., 0]
    G.FusedAdamW([plain], lr=0.1).step()
    G.FusedAdamW([turned], lr=0.1).step()
    G.FusedAdamW([spread], lr=0.1).step()
    assert torch.equal(plain, turned) and torch.equal(plain, spread)
    wide = torch.nn.Parameter(torch.zeros(1, 30, device="cuda"))
    wide.grad = torch.ones(1, 1, device="cuda").expand(1, 30)
    G.FusedAdamW([wide], lr=0.1).step()
    assert (wide.unique().numel() == 1) and float(wide[0, 0]) < 0
    cut = torch.nn.Parameter(torch.zeros(8, 8, device="cuda")[:, :4])
    cut.grad = torch.zeros(8, 4, device="cuda")
    with pytest.raises(_lib.GcpnetHipError, match="fill its memory"):
        G.FusedAdamW([cut]).step()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_infinities_and_nans_stay_where_they_are(bits):
    p, g = start(1000)
    p.grad.copy_(gradient(p, g) + 0.01)
    p.grad[7], p.grad[300], p.grad[999] = math.inf, math.nan, -math.inf
    opt = G.FusedAdamW([p], lr=1e-2, state_bits=bits)
    for _ in range(3):
        opt.step()
    bad = torch.zeros(1000, dtype=torch.bool)
    bad[[7, 300, 999]] = True
    for x in (p.detach(), opt.state[p]["exp_avg"].float(), opt.state[p]["exp_avg_sq"].float()):
        assert torch.equal(~torch.isfinite(x.cpu()), bad)


@pytest.mark.gpu
def test_stochastic_rounding_is_unbiased():
    """Without gradients v shrinks by 1 - b2 a step, far less than half the distance of two codes: the mean has to follow all the
    same.  A code is at most v / 8 from the next, so a step adds a standard deviation of at most v / 16, 50 steps 0.45 v, the mean of
    2^20 elements 4.4e-4 v; within six of them, 2.7e-3."""
    n = 1 << 20
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    p.grad = torch.randn(n, generator=torch.Generator().manual_seed(0)).cuda()
    opt = G.FusedAdamW([p], state_bits=8, lr=0.0, weight_decay=0.0)
    opt.step()
    st = opt.state[p]
    value = lambda: decode(st["exp_avg_sq"].cpu().view(torch.uint8), st["exp_avg_sq_scale"].cpu()).double()  # noqa: E731
    first = value()
    p.grad.zero_()
    for _ in range(50):
        opt.step()
    last = value()
    big = first > first.view(-1, 256).amax(1, keepdim=True).expand(-1, 256).reshape(-1) * 2.0 ** -10  # (no element at the smallest code)
    ratio = float(last[big].sum() / first[big].sum())
    assert abs(ratio - 0.999 ** 50) < 2.7e-3 * 2
    assert (last[first > 0] > 0).all()


@pytest.mark.gpu
def test_master_copies():
    """bf16 parameters move by steps far below their own rounding; a parameter that was written from outside starts from there."""
    p = torch.nn.Parameter(torch.ones(300, device="cuda", dtype=torch.bfloat16))
    p.grad = torch.ones_like(p)
    opt = G.FusedAdamW([p], lr=1e-4, weight_decay=0.0)
    for _ in range(40):  # 40 steps of 1e-4: one step is 1/78 of the distance of two bf16 numbers below 1
        opt.step()
    assert abs(float(opt.state[p]["master"][0]) - (1 - 40e-4)) < 1e-5 and float(p[0]) == float(torch.tensor(1 - 40e-4).bfloat16())
    with torch.no_grad():
        p[:100] = 3.0
    opt.step()
    m = opt.state[p]["master"]
    assert abs(float(m[0]) - (3 - 1e-4)) < 1e-5 and abs(float(m[200]) - (1 - 41e-4)) < 1e-5


@pytest.mark.gpu
def test_a_captured_step_counts_on():
    """step() inside a hipGraph: replays equal eager steps bit for bit (moments in 8 bits, clipping, changing gradients)."""
    def build():
        ps = [start(n, d) for n, d in ((5000, torch.float32), (777, torch.bfloat16), (12, torch.float32))]
        return ps, G.FusedAdamW([p for p, _ in ps], lr=1e-2, state_bits=8, max_grad_norm=1.0, seed=9)

    a, oa = build()
    b, ob = build()
    draws = [[gradient(p, g) for p, g in a] for _ in range(6)]

    def feed(ps, k):
        for (p, _), x in zip(ps, draws[k]):
            p.grad.copy_(x)

    with pytest.raises(RuntimeError, match="eager step before capturing"):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ob.step()
    b, ob = build()
    for k in range(2):
        feed(a, k)
        oa.step()
        feed(b, k)
        ob.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ob.step()
    for k in range(2, 6):
        feed(a, k)
        oa.step()
        feed(b, k)
        graph.replay()
        torch.cuda.synchronize()
        assert float(oa.grad_norm) == float(ob.grad_norm)
        for (p, _), (q, _) in zip(a, b):
            assert torch.equal(p, q)
            for key, v in oa.state[p].items():
                w = ob.state[q][key]
                assert torch.equal(v.view(torch.uint8), w.view(torch.uint8)) if v.dtype == E4M3 else torch.equal(v, w), key


@pytest.mark.gpu
def test_another_stream_and_the_version_counter():
    p, g = start(10000)
    q = torch.nn.Parameter(p.detach().clone())
    p.grad.copy_(gradient(p, g))
    q.grad = p.grad.clone()
    G.FusedAdamW([p], lr=0.1).step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    before = q._version
    with torch.cuda.stream(side):
        G.FusedAdamW([q], lr=0.1).step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(p, q) and q._version > before


@pytest.mark.gpu
def test_more_than_2_to_the_32_elements():
    """One bf16 tensor of 2^32 + 300 elements with 8-bit moments: its last 300 elements, whose indices need a 33rd bit."""
    if torch.cuda.get_device_properties(0).total_memory < 100 << 30:
        pytest.skip("needs 60 GiB of GPU memory")
    n, tail = (1 << 32) + 300, 300
    p = torch.nn.Parameter(torch.zeros(n, device="cuda", dtype=torch.bfloat16))
    p.grad = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    gr = torch.randn(tail, generator=torch.Generator().manual_seed(0)).bfloat16()
    p.grad[-tail:] = gr.cuda()
    opt = G.FusedAdamW([p], lr=1e-2, state_bits=8, weight_decay=0.0)
    opt.step()
    st = opt.state[p]
    g = gr.float()
    f = torch.float32
    m1, v1 = g * torch.tensor(1 - 0.9, dtype=f), (g * torch.tensor(1 - 0.999, dtype=f)) * g
    cm, cv, sm, sv = encode(m1, v1, 1, first=1 << 32)
    assert torch.equal(st["exp_avg"][-tail:].view(torch.uint8).cpu(), cm) and torch.equal(st["exp_avg_sq"][-tail:].view(torch.uint8).cpu(), cv)
    assert torch.equal(st["exp_avg_scale"][-2:].cpu(), sm) and torch.equal(st["exp_avg_sq_scale"][-2:].cpu(), sv)
    check_update(st["master"][-tail:].cpu(), m1, v1, torch.zeros(tail), g, torch.zeros(tail), torch.zeros(tail), 1, 1e-2, 0.9, 0.999, 1e-8, 0.0)
    assert float(st["master"][:1 << 20].abs().max()) == 0.0
    del p, opt, st
    torch.cuda.empty_cache()


@pytest.mark.gpu
def test_shared_memory_is_refused():
    a = torch.nn.Parameter(torch.zeros(600, device="cuda"))
    b = torch.nn.Parameter(a.detach()[300:])
    c = torch.nn.Parameter(torch.zeros(5, device="cuda"))
    for p in (a, b, c):
        p.grad = torch.ones_like(p)
    with pytest.raises(_lib.GcpnetHipError, match="share memory"):
        G.FusedAdamW([c, a, b]).step()
    whole = torch.zeros(600, device="cuda")  # (side by side is no overlap)
    halves = [torch.nn.Parameter(whole[:300]), torch.nn.Parameter(whole[300:])]
    for p in halves:
        p.grad = torch.ones_like(p)
    G.FusedAdamW(halves, lr=0.5, weight_decay=0.0).step()
    # the first step is -lr g / (|g| + eps): the root, the reciprocal and the corrections are off by a few units of 2^-24 each
    assert torch.allclose(whole, torch.full_like(whole, -0.5), rtol=1e-6, atol=0)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_state_whose_memory_moved(bits):
    """A state tensor whose data lie elsewhere since the last step is read and written where it is now."""
    def run(move):
        p = torch.nn.Parameter(torch.linspace(-1, 1, 700, device="cuda"))
        opt = G.FusedAdamW([p], lr=1e-2, state_bits=bits)
        for k in range(4):
            p.grad = torch.linspace(1, 2, 700, device="cuda") * (k + 1)
            opt.step()
            if move:
                for v in opt.state[p].values():
                    old = v.data
                    v.data = old.clone()
                    (old if old.element_size() > 1 else old.view(torch.uint8)).zero_()
        return p.detach()

    assert torch.equal(run(False), run(True))
