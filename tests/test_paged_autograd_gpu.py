"""The attention operators under torch's differentiation: what they do not differentiate they refuse, and what they write
in place torch knows of."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

import libcertex_amd as certex
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu


def rand(*shape, dtype=torch.float32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + sum(shape))
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def cache():
    pool, table = torch.zeros((3, 8, 2, 64), device="cuda"), torch.zeros((5, 3), dtype=torch.int32, device="cuda")
    return pool, table, torch.arange(5, dtype=torch.int32, device="cuda")


def test_tangents_are_refused(gpu):
    """Forward-mode differentiation of any tensor is an error, whether or not it asks for a gradient too; without a tangent,
    and with forward mode switched off, the calls are as ever."""
    rope = certex.Rotary(64)
    pool, table, p = cache()
    x, scores, ids, values = rand(5, 2, 64), rand(2, 1, 4), torch.zeros((2, 1, 4), dtype=torch.int64, device="cuda"), rand(2, 9, 64)
    plain = rope(x, p)
    with fwd.dual_level():
        def dual(t, grad=False):
            return fwd.make_dual(t.clone().requires_grad_(grad), torch.ones_like(t))

        calls = [
            lambda: rope(dual(x), p), lambda: rope(dual(x, True), p), lambda: rope(dual(x), p, transpose=True),
            lambda: rope(x, p, out=dual(x)), lambda: rope(dual(x)[..., ::2].repeat(1, 1, 2), p),
            lambda: certex.append_pages(dual(x), x, pool, pool.clone(), table, p),
            lambda: certex.append_pages(x, dual(x), pool, pool.clone(), table, p),
            lambda: certex.append_pages(x, x, dual(pool), pool.clone(), table, p),
            lambda: certex.append_pages(x, x, pool, dual(pool), table, p),
            lambda: certex.append_pages(x, x, pool, pool.clone(), table, p, q=dual(x)),
            lambda: certex.paged_attention(dual(x), pool, pool, table, p),
            lambda: certex.paged_attention(x, dual(pool), pool, table, p),
            lambda: certex.paged_attention(x, pool, dual(pool), table, p),
            lambda: certex.selected_attention(dual(scores), ids, values, 1.0),
            lambda: certex.selected_attention(scores, ids, dual(values), 1.0),
        ]
        for call in calls:
            with pytest.raises(ValueError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
                call()
        assert torch.equal(rope(x, p), plain)
        with fwd._set_fwd_grad_enabled(False):
            assert torch.equal(rope(fwd.make_dual(x, torch.ones_like(x)), p), plain)
        # the gradient of a dual tensor, which a backward pass rotates
        y = rope(x.clone().requires_grad_(), p)
        with pytest.raises(RuntimeError):
            y.backward(dual(x))
    assert (pool == 0).all()
