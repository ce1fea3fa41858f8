"""Attention with masks and bent scores in float64 on the CPU, and how far float32 computations may be from it."""

import torch

from tests.paged_reference import UNIT

U = 2.0**-24


def attend(q, positions, keys, values, scale, prefix=0, window=None, cap=None, slopes=None, there=None, weight=0.0,
           key_sizes=None, value_sizes=None):
    """Queries (n, heads, d) at `positions` (n,) over the keys (length, kv, d) and values of one sequence. Returns out (n, heads, dv),
    lse (n, heads) and bounds of their errors before the output is rounded.

    A weight w is off by e w: e is 4 (sqrt(d) + 4) u sum |scale q k| of the dot product and its scaling, as random roundings
    of d terms; 8 u (cap + slope distance + |y|) of the bent score, whose last operations round what is of that size, and
    4 u of the difference from the reference, of the exponential and of the weight, which `weight` adds to if weights are
    rounded again. An output of weights w / sum w is then off by sum w e |v| + (sum w e) |out|, and the two sums of n
    terms add 4 (sqrt(n) + 1) u of sum w |v| each. key_sizes and value_sizes: what |k| and |v| are where those are computed as
    sums of terms, the sizes of the terms."""
    q, keys, values = q.double().cpu(), keys.double().cpu(), values.double().cpu()
    n, heads, d = q.shape
    length, group = keys.shape[0], heads // keys.shape[1]
    p, t = positions.cpu()[:, None], torch.arange(length)
    seen = (t <= p) | (t < prefix)
    if window:
        seen &= t > p - window
    if there is not None:
        seen &= there[:length]
    out = torch.zeros((n, heads, values.shape[2]), dtype=torch.float64)
    lse = torch.full((n, heads), float("-inf"), dtype=torch.float64)
    out_room, lse_room = torch.zeros_like(out), torch.zeros_like(lse)
    if length == 0:
        return out, lse, out_room, lse_room
    key_sizes = keys.abs() if key_sizes is None else key_sizes
    value_sizes = values.abs() if value_sizes is None else value_sizes
    for h in range(heads):
        k, v = keys[:, h // group], values[:, h // group]
        used = seen.any(0)[:, None]
        k, v = torch.where(used, k, 0.0), torch.where(used, v, 0.0)
        k_size = torch.where(used, key_sizes[:, h // group], 0.0)
        v_size = torch.where(used, value_sizes[:, h // group], 0.0)
        x = scale * (q[:, h] @ k.T)
        size = abs(scale) * (q[:, h].abs() @ k_size.T)
        y = cap * torch.tanh(x / cap) if cap else x
        lean = float(slopes[h]) * (p - t).abs() if slopes is not None else torch.zeros(1, dtype=torch.float64)
        y = y - lean
        e = 4 * (d**0.5 + 4) * U * size + 4 * U + weight
        if cap or slopes is not None:
            e = e + 8 * U * ((cap or 0.0) + lean.abs() + y.abs())
        y = torch.where(seen, y, float("-inf"))
        some = seen.any(-1)
        w = torch.where(some[:, None], torch.softmax(y, -1), 0.0)
        out[:, h], lse[:, h] = w @ v, torch.logsumexp(y, -1)
        off = torch.where(seen, w * e, 0.0)
        sums = 4 * (length**0.5 + 1) * U
        out_room[:, h] = off @ v_size + off.sum(-1, keepdim=True) * out[:, h].abs() + 2 * sums * (w @ v_size)
        lse_room[:, h] = off.sum(-1) + sums + 8 * U * (1 + torch.where(some, lse[:, h].abs(), 0.0))
    return out, lse, out_room, lse_room


def check(got, got_lse, want):
    """An output of its type against attend's: half a unit in the last place more than the bound."""
    out, lse, out_room, lse_room = want
    unit = UNIT[got.dtype]
    bound = out_room + unit * (out.abs() + out_room) + torch.finfo(got.dtype).tiny
    err = (got.double().cpu() - out).abs()
    assert (err <= bound).all(), (float(err.max()), float((err / bound).max()))
    if got_lse is not None:
        got_lse, empty = got_lse.double().cpu(), lse.isinf()
        assert torch.equal(got_lse[empty], lse[empty])
        assert ((got_lse - lse).abs()[~empty] <= lse_room[~empty]).all(), float((got_lse - lse).abs()[~empty].max())
