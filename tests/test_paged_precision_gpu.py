"""How precise the attention operators are inside, where the rounding of their outputs does not hide it: values that
cancel, scores far from 0. Bounds are in units u = 2^-24, half a unit in the last place of float32."""

import pytest
import torch

import libcertex_amd as certex
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
U = 2.0**-24


def cancelling(weights, width, dtype, seed):
    """Values (rows, n, width) of a type whose sums under the softmax weights (rows, n) leave little of their terms: each
    value cancels the sum of those before it as far as the type goes."""
    g = torch.Generator().manual_seed(seed)
    rows, n = weights.shape
    v = torch.zeros((rows, n, width), dtype=torch.float64)
    v[:, 0] = (256 * (1 + torch.rand((rows, width), generator=g, dtype=torch.float64))).to(dtype).double()
    left = weights[:, :1] * v[:, 0]
    for t in range(1, n):
        v[:, t] = (-left / weights[:, t : t + 1]).to(dtype).double()
        left = left + weights[:, t : t + 1] * v[:, t]
    return v


@pytest.mark.parametrize("dtype", TYPES)
def test_attend_weights_are_whole(gpu, dtype):
    """The softmax's weights enter the product with the values as float32 has them. Scores are exact, |scale score| <= 1:
    a weight is off by 5 u of its exponent (|x| <= 1.5 and differences to 2.9 in powers of 2, rounded three times), 2 u of
    the exponential and u of its own; 8 u are for the sums."""
    b, h, d, n = 32, 4, 64, 4
    g = torch.Generator().manual_seed(1)
    s = torch.randint(-128, 129, (b, h, n), generator=g) / 128.0
    w = torch.softmax(s.double(), -1)
    v = cancelling(w.reshape(b * h, n), d, dtype, 2).reshape(b, h, n, d)
    kp, vp = torch.zeros((b, 8, h, d), dtype=dtype), torch.zeros((b, 8, h, d), dtype=dtype)
    kp[:, :n, :, 0] = s.transpose(1, 2).to(dtype)
    vp[:, :n] = v.transpose(1, 2).to(dtype)
    q = torch.zeros((b, h, d), dtype=dtype)
    q[..., 0] = 1.0
    assert torch.equal(kp[:, :n, :, 0].double(), s.transpose(1, 2).double()) and torch.equal(vp[:, :n].double(), v.transpose(1, 2))
    table = torch.arange(b, dtype=torch.int32).view(b, 1)
    out = certex.paged_attention(q.cuda(), kp.cuda(), vp.cuda(), table.cuda(),
                                 torch.full((b,), n, device="cuda"), scale=1.0).double().cpu()
    want, spread = (w[..., None] * v).sum(2), (w[..., None] * v.abs()).sum(2)
    bound = 16 * U * spread + (ref.UNIT[dtype] + 16 * U) * want.abs() + ref.UNIT[dtype] * torch.finfo(dtype).tiny
    assert (want.abs() < spread / 1000).all()  # the output's own rounding hides nothing
    assert ((out - want).abs() <= bound).all(), float(((out - want).abs() / bound).max())
