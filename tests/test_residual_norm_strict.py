"""The comparisons of test_residual_norm once more, with a NaN where none belongs counted as an error."""
import math

import pytest
import torch

from tests import test_residual_norm as R


def strict(out, want, what=""):
    for k, (v, tol) in want.items():
        got = out[k].detach().cpu().double()
        assert got.shape == v.shape, (k, got.shape)
        assert torch.isfinite(v).all() and torch.isfinite(tol).all(), k
        kind = torch.finfo(out[k].dtype)
        tol = tol + kind.smallest_normal * kind.eps / 2
        good = (got - v).abs() <= tol  # (False for NaN)
        # a value from max + half a step on rounds to infinity
        good |= torch.isinf(got) & (got.sign() == v.sign()) & (v.abs() + tol >= kind.max)
        assert good.all(), f"{what} {k}: {int((~good).sum())} of {v.numel()} off or NaN"


def test_a_nan_is_an_error():
    v = torch.ones(3, 4)
    want = {"s": (v.double(), 0 * v.double())}
    strict({"s": v}, want)
    for bad in (math.nan, math.inf, -math.inf, 1.5):
        w = v.clone()
        w[1, 2] = bad
        with pytest.raises(AssertionError):
            strict({"s": w}, want)
    top = torch.tensor([65504.0], dtype=torch.float16)
    strict({"s": top * 2}, {"s": (top.double() + 16, torch.zeros(1).double())})  # (rounds to infinity)


@pytest.fixture
def strictly(monkeypatch):
    monkeypatch.setattr(R, "compare", strict)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,d", R.SHAPES)
def test_sizes(strictly, rows, d, t):
    R.test_sizes(rows, d, t)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("pre", [None, "layer", "rms"])
@pytest.mark.parametrize("post", [None, "layer", "rms"])
@pytest.mark.parametrize("gate,gact", [(None, None), ("channel", None), ("channel", "silu"), ("element", "sigmoid"), ("element", "leakyrelu")])
def test_forms(strictly, gate, gact, post, pre, t):
    R.test_forms(gate, gact, post, pre, t)


@pytest.mark.gpu
@pytest.mark.parametrize("wt", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("rows,d", [(9000, 40), (2100, 1000), (1100, 2044), (1100, 4096), (600, 6000), (300, 16000)])
def test_many_rows(strictly, rows, d, wt):
    R.test_many_rows(rows, d, wt)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_strided_rows(strictly, t):
    R.test_strided_rows_and_leading_dimensions(t)


@pytest.mark.gpu
@pytest.mark.parametrize("off", [1, 4, 8])
def test_addresses_off_16_bytes(strictly, off):
    R.test_addresses_off_16_bytes(off)
