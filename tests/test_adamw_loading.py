"""FusedAdamW: state that does not fit is refused before anything has changed, and tables of a step follow their parameters' layout."""
import copy

import pytest
import torch

import gcpnet_amd as G
from gcpnet_amd import _lib
from gcpnet_amd.optim import _Part

E4M3 = torch.float8_e4m3fn


def state8(p, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = p.numel()
    blocks = -(-n // 256)
    like = lambda: torch.empty_like(p, dtype=torch.float32)  # noqa: E731
    return dict(step=torch.tensor(3.0), exp_avg=like().copy_(torch.randn(p.shape, generator=g)).to(E4M3), exp_avg_sq=like().copy_(torch.rand(p.shape, generator=g)).to(E4M3),
                exp_avg_scale=2.0 ** torch.arange(blocks), exp_avg_sq_scale=0.5 ** torch.arange(blocks))


def values(t, scale):
    """Moments as they are meant: every code times the scale of its 256 elements in memory order."""
    codes = t.as_strided((t.numel(),), (1,)).float()
    out = torch.empty_like(t, dtype=torch.float32)
    out.as_strided((t.numel(),), (1,)).copy_(codes * scale.repeat_interleave(256)[:t.numel()])
    return out


def snapshot(opt):
    return copy.deepcopy([{k: v for k, v in g.items() if k != "params"} for g in opt.param_groups]), {
        p: (st, {k: (v, v.clone() if torch.is_tensor(v) else v) for k, v in st.items()}) for p, st in opt.state.items()}


def assert_unchanged(opt, before):
    groups, state = before
    assert [{k: v for k, v in g.items() if k != "params"} for g in opt.param_groups] == groups
    assert list(opt.state) == list(state)
    for p, (st, held) in state.items():
        assert opt.state[p] is st and st.keys() == held.keys()
        for k, (v, was) in held.items():
            assert st[k] is v and (not torch.is_tensor(v) or (v.dtype == was.dtype and torch.equal(v.float(), was.float())))


def refuses(opt, saved, error, match):
    before = snapshot(opt)
    with pytest.raises(error, match=match):
        opt.load_state_dict(saved)
    assert_unchanged(opt, before)


# ---------------------------------------------------------------------------------------------------------------- layouts of 8-bit state
@pytest.mark.parametrize("shape", [(40, 30), (6, 5, 4, 7), (3, 1, 300)])
def test_codes_keep_their_scales_or_are_refused(shape):
    """The scales of 8-bit moments go by the memory order: codes are taken over where that is the same, and refused where it is not."""
    plain = torch.zeros(shape)
    turned = torch.zeros(shape[::-1]).permute(*range(len(shape))[::-1])
    for a in (plain, turned):
        for b in (plain, turned):
            p, q = torch.nn.Parameter(a.clone()), torch.nn.Parameter(b.clone())
            o1, o2 = G.FusedAdamW([p], state_bits=8), G.FusedAdamW([q], state_bits=8)
            o1.state[p] = state8(p)
            want = [values(o1.state[p][k], o1.state[p][k + "_scale"]) for k in ("exp_avg", "exp_avg_sq")]
            same = a is b
            if same:
                o2.load_state_dict(o1.state_dict())
                got = [values(o2.state[q][k], o2.state[q][k + "_scale"]) for k in ("exp_avg", "exp_avg_sq")]
                assert all(torch.equal(x, y) for x, y in zip(got, want))
            else:
                refuses(o2, o1.state_dict(), _lib.GcpnetHipError, "memory order")


def test_one_block_and_unit_dimensions_load_in_any_layout():
    for shape in ((16, 16), (1, 900), (900, 1, 1)):  # (all elements share a scale, or there is one order only)
        p = torch.nn.Parameter(torch.zeros(shape))
        q = torch.nn.Parameter(torch.zeros(shape[::-1]).permute(*range(len(shape))[::-1]))
        o1, o2 = G.FusedAdamW([p], state_bits=8), G.FusedAdamW([q], state_bits=8)
        o1.state[p] = state8(p)
        o2.load_state_dict(o1.state_dict())
        for k in ("exp_avg", "exp_avg_sq"):
            assert torch.equal(values(o1.state[p][k], o1.state[p][k + "_scale"]), values(o2.state[q][k], o2.state[q][k + "_scale"]))


# ---------------------------------------------------------------------------------------------------------------- refused loads
def test_a_refused_load_changes_nothing():
    a, b = torch.nn.Parameter(torch.zeros(5, 70)), torch.nn.Parameter(torch.zeros(5, 70))
    o1, o2 = G.FusedAdamW([a], state_bits=8, lr=0.5, seed=4), G.FusedAdamW([b], state_bits=32, lr=0.25, seed=6)
    o1.state[a] = state8(a)
    o2.state[b] = dict(step=torch.tensor(2.0), exp_avg=torch.randn(5, 70), exp_avg_sq=torch.rand(5, 70))
    wrong = o1.state_dict()
    wrong["param_groups"][0]["state_bits"] = 32  # (codes, said to be fp32 moments)
    refuses(o2, wrong, _lib.GcpnetHipError, "state_bits=32")
    short = o1.state_dict()
    short["state"] = {0: dict(short["state"][0], exp_avg_scale=torch.ones(1))}
    refuses(o2, short, _lib.GcpnetHipError, "contiguous scales")
    other = G.FusedAdamW([torch.nn.Parameter(torch.zeros(3)), torch.nn.Parameter(torch.zeros(3))])
    refuses(o2, other.state_dict(), ValueError, "size")  # (torch's own refusal: another number of parameters)
    options = o2.state_dict()
    options["param_groups"][0]["betas"] = (1.0, 0.9)
    refuses(o2, options, ValueError, "betas")


def test_the_last_parameter_refused_leaves_the_first_alone():
    ps = [torch.nn.Parameter(torch.zeros(n)) for n in (4, 5)]
    fresh = lambda: dict(step=torch.tensor(1.0), exp_avg=torch.ones(1), exp_avg_sq=torch.ones(1))  # noqa: E731
    opt = G.FusedAdamW(ps)
    saved = opt.state_dict()
    saved["state"] = {0: dict(fresh(), exp_avg=torch.ones(4), exp_avg_sq=torch.ones(4)), 1: dict(fresh(), exp_avg=torch.ones(6), exp_avg_sq=torch.ones(6))}
    refuses(opt, saved, _lib.GcpnetHipError, "shape")


def test_groups_without_own_options_keep_theirs():
    """A torch.optim.AdamW state knows neither state_bits nor seed: each group keeps its own, and fp32 moments are refused for 8 bits."""
    ps = [torch.nn.Parameter(torch.randn(4)) for _ in range(2)]
    theirs = torch.optim.AdamW([dict(params=ps[:1]), dict(params=ps[1:])], lr=0.1)
    opt = G.FusedAdamW([dict(params=ps[:1], seed=9), dict(params=ps[1:], state_bits=8, seed=11)], seed=3)
    opt.load_state_dict(theirs.state_dict())  # (no state yet: only options)
    assert [(g["state_bits"], g["seed"], g["lr"]) for g in opt.param_groups] == [(32, 9, 0.1), (8, 11, 0.1)]
    for p in ps:
        p.grad = torch.ones_like(p)
    theirs.step()
    refuses(opt, theirs.state_dict(), _lib.GcpnetHipError, "state_bits=8")


@pytest.mark.parametrize("option", [dict(maximize=True), dict(amsgrad=True), dict(differentiable=True)])
def test_state_of_another_update_is_refused(option):
    p, q = torch.nn.Parameter(torch.randn(4)), torch.nn.Parameter(torch.randn(4))
    theirs = torch.optim.AdamW([p], **option)
    opt = G.FusedAdamW([q])
    refuses(opt, theirs.state_dict(), ValueError, next(iter(option)))
    with pytest.raises(ValueError, match=next(iter(option))):
        G.FusedAdamW([dict(params=[q], **option)])
    opt.param_groups[0].update(option)
    with pytest.raises(ValueError, match=next(iter(option))):
        opt.step()


def test_coupled_decay_is_refused():
    p, q = torch.nn.Parameter(torch.randn(4)), torch.nn.Parameter(torch.randn(4))
    refuses(G.FusedAdamW([q]), torch.optim.Adam([p], weight_decay=0.1).state_dict(), ValueError, "decoupled")
    opt = G.FusedAdamW([q])
    opt.load_state_dict(torch.optim.Adam([p], weight_decay=0.0).state_dict())  # (without decay they are the same)
    assert opt.param_groups[0]["weight_decay"] == 0.0


def test_hooks_of_a_load_see_and_change_what_is_loaded():
    p, q = torch.nn.Parameter(torch.zeros(300)), torch.nn.Parameter(torch.zeros(300))
    o1, o2 = G.FusedAdamW([p], state_bits=8), G.FusedAdamW([q], state_bits=8)
    o1.state[p] = state8(p)

    def before(opt, saved):
        st = {0: dict(saved["state"][0], step=torch.tensor(40.0))}
        return dict(saved, state=st)

    seen = []
    o2.register_load_state_dict_pre_hook(before)
    o2.register_load_state_dict_post_hook(lambda opt: seen.append(opt.state[q]["exp_avg"].dtype))
    o2.load_state_dict(o1.state_dict())
    assert float(o2.state[q]["step"]) == 40.0 and seen == [E4M3]
    assert float(o1.state[p]["step"]) == 3.0


# ---------------------------------------------------------------------------------------------------------------- steps
def test_tables_go_by_the_strides():
    """A parameter turned at its address, with a gradient of the new shape, does not match the old table."""
    p = torch.nn.Parameter(torch.zeros(4, 6))
    st = dict(step=torch.tensor(0.0), exp_avg=torch.zeros(4, 6), exp_avg_sq=torch.zeros(4, 6))
    g = torch.ones(4, 6)
    part = _Part(0, torch.float32, [(p, g, st, 0)], 32)
    assert G.FusedAdamW._same(part, [g]) and G.FusedAdamW._same(part, [g.clone()])
    p.data = p.data.t()
    assert not G.FusedAdamW._same(part, [torch.ones(6, 4)])


@pytest.mark.gpu
def test_a_parameter_turned_between_two_steps_is_refused():
    p = torch.nn.Parameter(torch.zeros(40, 30, device="cuda"))
    opt = G.FusedAdamW([p])
    p.grad = torch.ones_like(p)
    opt.step()
    p.grad = None
    p.data = p.data.t()
    p.grad = torch.ones(30, 40, device="cuda")
    with pytest.raises(_lib.GcpnetHipError, match="shape and strides"):
        opt.step()


def test_a_tensor_of_more_workgroups_than_a_launch_takes():
    """2^24 workgroups of 256 threads are 2^32: refused on the host, for the update (4096 elements each) and for the norm (16384)."""
    lib = _lib.load()
    arr = (_lib.AdamWTensor * 1)()
    for name in ("param", "grad", "exp_avg", "exp_avg_sq", "step"):
        setattr(arr[0], name, 4096)
    arr[0].n = 4096 * ((1 << 24) - 1) + 1
    assert lib.gcpnet_adamw_step(1, arr, 0, 32, 1e-3, 0.9, 0.999, 1e-8, 0.0, 4096, None, 0, None) == -2
    arr[0].n = 16384 * ((1 << 24) - 1) + 1
    assert lib.gcpnet_grad_norm(1, arr, 0, 4096, None) == -2


def test_the_norm_of_no_gradients_is_zero():
    p = torch.nn.Parameter(torch.zeros(4))
    opt = G.FusedAdamW([p], max_grad_norm=1.0)
    opt.grad_norm = torch.tensor(7.0)  # (of a step before)
    opt.step()
    assert float(opt.grad_norm) == 0.0


@pytest.mark.gpu
def test_a_step_without_gradients_leaves_no_old_norm():
    p = torch.nn.Parameter(torch.zeros(4, device="cuda"))
    opt = G.FusedAdamW([p], max_grad_norm=1.0)
    p.grad = torch.full_like(p, 2.0)
    opt.step()
    assert abs(float(opt.grad_norm) - 4.0) < 1e-6
    p.grad = None
    opt.step()
    assert float(opt.grad_norm) == 0.0 and opt.grad_norm.device == p.device


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_run_goes_on_from_its_state_dict(dtype, bits):
    """Three steps, a state_dict, and three more steps of a new optimizer over the same tensors: bit for bit the six steps of one."""
    def run(reload):
        g = torch.Generator().manual_seed(0)
        ps = [torch.nn.Parameter(torch.randn(s, generator=g).to(dtype).cuda()) for s in ((40, 30), (7,))]
        ps.append(torch.nn.Parameter(torch.randn(30, 40, generator=g).to(dtype).cuda().t()))
        opt = G.FusedAdamW(ps, lr=1e-2, state_bits=bits, seed=5, max_grad_norm=1.0)
        for k in range(6):
            for p in ps:
                p.grad = torch.randn(p.shape, generator=g).to(dtype).cuda()
            if reload and k == 3:
                saved = copy.deepcopy(opt.state_dict())
                opt = G.FusedAdamW(ps, lr=1.0, state_bits=bits, max_grad_norm=1.0)
                opt.load_state_dict(saved)
            opt.step()
        return ps

    for a, b in zip(run(False), run(True)):
        assert torch.equal(a, b)
