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
@pytest.mark.parametrize("lo, hi", [(1e-30, 1e-3), (1e-3, 0.3), (0.3, 0.6), (0.59, 0.61), (0.6, 1.0), (0.79, 0.81), (1.0, 2.0), (2.0, 9.1), (9.0, 1e30)])
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


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("operator", ["paged", "prompt", "packed"])
@pytest.mark.parametrize("cap", [5.0, 50.0, 64.0, 1000.0])
def test_capped_scores(gpu, operator, dtype, cap):
    """cap tanh(x / cap) of one position in every type, small beside the cap and not: 3 units of tanh, and a rounding of 1 / cap, of its
    product with x (neither weighs more in tanh than in its argument) and of the product with cap, half a unit each of what may be a
    unit of half the size: 6 units in the last place."""
    heads = 30_000
    key = torch.zeros(1, 8, 1, 64, device="cuda", dtype=dtype)
    key[..., 0] = 1
    q = torch.zeros(1, heads, 64, device="cuda", dtype=dtype)
    q[0, :, 0] = (torch.logspace(-4, 2.5, heads, device="cuda") * torch.where(torch.arange(heads, device="cuda") % 2 == 0, 1, -1)).to(dtype)
    how = dict(scale=1.0, cap=cap, return_lse=True)
    if operator == "packed":
        # elements of 0 and 1 are held exactly, as codes 0 and 15 of a scale that float16 rounds: the key is what the pages hold
        pages = certex.PackedPages(1, 8, 1, 64)
        pages.append(key[:, 0], key[:, 0], ints([[0]]), ints([0]))
        x = q[0, :, 0].double() * pages.read(ints([[0]]), ints([0]), dtype=torch.float32)[0][0, 0, 0].double()
        lse = pages.attend(q, ints([[0]]), ints([1]), **how)[1]
    else:
        x = q[0, :, 0].double()
        if operator == "paged":
            lse = certex.paged_attention(q, key, key, ints([[0]]), ints([1]), **how)[1]
        else:
            lse = certex.prompt_attention(q, key, key, ints([[0]]), ints([1]), ints([0, 1]), **how)[1]
    want = cap * torch.tanh(x / cap)
    unit = 2.0 ** (torch.frexp(want)[1] - 24).double()
    assert float(((lse[0].double() - want).abs() / unit).max()) <= (8.0 if operator == "packed" else 6.0)  # (packed: its product's, too)
