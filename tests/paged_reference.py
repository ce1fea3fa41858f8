"""The attention operators' definitions in float64 on the CPU, and how far float32 computations with one
rounding at the end may be from them."""

import torch

UNIT = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}  # half a unit in the last place
# the softmax's weights enter the matrix product in float32, rounded to float16, or as a pair of
# bfloat16 (value and remainder)
WEIGHT = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-15}


def rotate(x, positions, frequencies, layout, rotary_dim, magnitude=1.0, transpose=False):
    """float64 (..., tokens, heads, dim)."""
    x = x.double().cpu()
    angle = positions.double().cpu()[..., None, None] * frequencies.double().cpu()
    c, s = magnitude * angle.cos(), magnitude * angle.sin() * (-1.0 if transpose else 1.0)
    y = x.clone()
    r = rotary_dim
    first, second = (slice(0, r // 2), slice(r // 2, r)) if layout == "half" else (slice(0, r, 2), slice(1, r, 2))
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * c - b * s, a * s + b * c
    return y


def assert_rotated(y, x, want, layout, rotary_dim, magnitude=1.0):
    """|error| <= u |y| + 16 2^-24 m (|a| + |b|): the angle is within pi 2^-24, sin and cos within 4 2^-24, the
    magnitude and the products round once each."""
    got, x = y.double().cpu(), x.double().cpu().abs()
    r = rotary_dim
    both = torch.zeros_like(x)
    first, second = (slice(0, r // 2), slice(r // 2, r)) if layout == "half" else (slice(0, r, 2), slice(1, r, 2))
    both[..., first] = both[..., second] = x[..., first] + x[..., second]
    # values below the type's smallest normal are rounded to a fixed spacing
    tiny = torch.finfo(y.dtype).tiny * UNIT[y.dtype]
    bound = UNIT[y.dtype] * want.abs() + 16 * 2.0**-24 * magnitude * both + tiny
    assert ((got - want).abs() <= bound).all(), float(((got - want).abs() - bound).max())
    assert torch.equal(y[..., r:].cpu(), y[..., r:].cpu()) and torch.equal(got[..., r:], want[..., r:])


def attend(q, keys, values, scale):
    """One query row of one sequence in float64: q (heads, d), keys (n, kv, d), values (n, kv, dv). Returns out
    (heads, dv), lse (heads,), and what bounds the error: sum of w |v|, and the largest sum of scale |q k|."""
    q, keys, values = q.double().cpu(), keys.double().cpu(), values.double().cpu()
    h, kv = q.shape[0], values.shape[1]
    g = h // kv
    if keys.shape[0] == 0:
        z = torch.zeros(h, values.shape[2], dtype=torch.float64)
        return z, torch.full((h,), float("-inf"), dtype=torch.float64), z, torch.zeros(h, dtype=torch.float64)
    out, lse, spread, dots = [], [], [], []
    for i in range(h):
        k, v = keys[:, i // g], values[:, i // g]
        s = scale * (k @ q[i])
        w = torch.softmax(s, 0)
        out.append(w @ v)
        lse.append(torch.logsumexp(s, 0))
        spread.append(w @ v.abs())
        dots.append((abs(scale) * (k.abs() @ q[i].abs())).max())
    return torch.stack(out), torch.stack(lse), torch.stack(spread), torch.stack(dots)


def assert_attended(got, want, spread, dots, n, d, lse=None, want_lse=None):
    """|error| <= u |out| + 2 e sum w |v|, e the relative error of a weight: of its exponent (rounding of the d-term dot
    product and of its scaling, as random roundings: 4 sqrt(d) 2^-24 sum |q k|, and of the exponential's argument:
    2^-22 of at most twice that sum), its own rounding, and 4 sqrt(n) 2^-24 of the sums over n positions."""
    e = 4 * (max(1, d) ** 0.5 + 4) * 2.0**-24 * dots + 4 * (max(1, n) ** 0.5 + 1) * 2.0**-24 + WEIGHT[got.dtype]
    bound = UNIT[got.dtype] * want.abs() + 2 * e[..., None] * spread + torch.finfo(got.dtype).tiny
    err = (got.double().cpu() - want).abs()
    assert (err <= bound).all(), (float(err.max()), float((err / bound).max()))
    if lse is not None:
        lse = lse.double().cpu()
        empty = want_lse.isinf()
        assert torch.equal(lse[empty], want_lse[empty])
        slack = (e + 2.0**-22 * (1 + want_lse.abs()))[~empty]
        assert ((lse - want_lse).abs()[~empty] <= slack).all()
