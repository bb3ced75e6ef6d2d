"""FusedAdamW: which state a load takes, and which it refuses."""
import copy

import pytest
import torch

import gcpnet_amd as G
from gcpnet_amd import _lib

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
                with pytest.raises(_lib.GcpnetHipError, match="memory order"):
                    o2.load_state_dict(o1.state_dict())


def test_one_block_and_unit_dimensions_load_in_any_layout():
    for shape in ((16, 16), (1, 900), (900, 1, 1)):  # (all elements share a scale, or there is one order only)
        p = torch.nn.Parameter(torch.zeros(shape))
        q = torch.nn.Parameter(torch.zeros(shape[::-1]).permute(*range(len(shape))[::-1]))
        o1, o2 = G.FusedAdamW([p], state_bits=8), G.FusedAdamW([q], state_bits=8)
        o1.state[p] = state8(p)
        o2.load_state_dict(o1.state_dict())
        for k in ("exp_avg", "exp_avg_sq"):
            assert torch.equal(values(o1.state[p][k], o1.state[p][k + "_scale"]), values(o2.state[q][k], o2.state[q][k + "_scale"]))


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
