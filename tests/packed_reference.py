"""What 4-bit pages hold, from the definition: codes, scales and offsets of groups of 64 elements, on the CPU."""

import torch

GROUP, MOST, FIFTEENTH = 64, 65504.0, torch.tensor(1 / 15, dtype=torch.float32)


def quantise(x):
    """x (..., d): codes (..., d) as float64, and every element's scale and offset (float64)."""
    x = x.cpu()
    code, scale, offset = (torch.empty(x.shape, dtype=torch.float64) for _ in range(3))
    for at in range(0, x.shape[-1], GROUP):
        part = x[..., at : at + GROUP]
        low = part.float().amin(-1, keepdim=True).clamp(-MOST, MOST).half()
        step = ((part.float().amax(-1, keepdim=True) - low.float()) * FIFTEENTH).clamp(0, MOST).half()
        o, s = low.double(), step.double()
        c = torch.where(s > 0, ((part.double() - o) / torch.where(s > 0, s, 1.0)).round().clamp(0, 15), 0.0)
        nan = part.isnan().any(-1, keepdim=True)
        code[..., at : at + GROUP] = torch.where(nan, 0.0, c)
        scale[..., at : at + GROUP] = torch.where(nan, float("nan"), s)
        offset[..., at : at + GROUP] = torch.where(nan, float("nan"), o)
    return code, scale, offset


def stored(x):
    """What the pages hold of x, and the sizes of the two terms it is the sum of (float64)."""
    code, scale, offset = quantise(x)
    return offset + scale * code, offset.abs() + scale * code
