"""The cap of attention scores against tanh in float64: how far the operators' float32 form is off, in units in the last place."""

import pytest
import torch

import libcertex_amd as certex
from tests.test_paged_gpu import ints

pytestmark = pytest.mark.gpu


def capped(u, operator):
    """tanh(u) as the operator takes it: the logarithm of one position's weight, whose key is 1, with a cap and a scale of 1."""
    out = []
    key = torch.zeros(1, 8, 1, 8, device="cuda")
    key[..., 0] = 1
    for part in u.split(60_000):
        q = torch.zeros(1, part.numel(), 8, device="cuda")
        q[0, :, 0] = part
        if operator == "paged":
            lse = certex.paged_attention(q, key, key, ints([[0]]), ints([1]), scale=1.0, cap=1.0, return_lse=True)[1]
        else:
            lse = certex.prompt_attention(q, key, key, ints([[0]]), ints([1]), ints([0, 1]), scale=1.0, cap=1.0, return_lse=True)[1]
        out.append(lse[0])
    return torch.cat(out)


@pytest.mark.parametrize("operator", ["paged", "prompt"])
@pytest.mark.parametrize("lo, hi", [(1e-30, 1e-3), (1e-3, 0.3), (0.3, 0.6), (0.59, 0.61), (0.6, 1.0), (1.0, 2.0), (2.0, 9.1), (9.0, 1e30)])
def test_tanh(gpu, operator, lo, hi):
    """3 units in the last place (derived where tanh_of is), on both sides of where its form changes and of 0."""
    g = torch.Generator(device="cuda").manual_seed(1)
    u = lo * (hi / lo) ** torch.rand(120_000, generator=g, device="cuda", dtype=torch.float64)
    u = torch.cat([u, torch.linspace(lo, min(hi, 20.0), 50_000, device="cuda", dtype=torch.float64)]).float()
    u = torch.where(torch.arange(u.numel(), device="cuda") % 2 == 0, u, -u)
    want = torch.tanh(u.double())
    got = capped(u, operator).double()
    unit = 2.0 ** (torch.frexp(want)[1] - 24).double()
    assert float(((got - want).abs() / unit).max()) <= 3.0


@pytest.mark.parametrize("operator", ["paged", "prompt"])
def test_tanh_ends(gpu, operator):
    u = torch.tensor([0.0, 1e-38, 15.0, 1e38, -1e38, float("nan")], device="cuda")
    got = capped(u, operator)
    assert got[:5].tolist() == [0.0, float(u[1]), 1.0, 1.0, -1.0] and got[5].isnan()
