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


def test_written_tensors_change_version(gpu):
    """A backward pass whose saved tensor the calls have written over since raises, as torch's in-place operators make it."""
    rope = certex.Rotary(64)
    pool, table, p = cache()
    w, x, buf = torch.ones((), device="cuda", requires_grad=True), rand(5, 2, 64), rand(5, 2, 64, seed=1)
    y = w * buf
    rope(x, p, out=buf)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    y = w * buf
    rope(buf, p, out=buf)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    k_pages, v_pages = pool.clone(), pool.clone()
    for saved in (k_pages, v_pages, k_pages.transpose(1, 2), v_pages[1:2]):  # a view shares its tensor's version
        y = w * saved
        certex.append_pages(x, x, k_pages, v_pages, table, p)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    # what is only read is not: these backward passes run
    before = [t._version for t in (x, k_pages, v_pages, buf)]
    certex.paged_attention(x, k_pages, v_pages, table, p)
    rope(x, p)
    certex.append_pages(x, x, pool.clone(), pool.clone(), table, p, rotary=rope, q=buf)
    assert before == [t._version for t in (x, k_pages, v_pages, buf)]
    with torch.inference_mode():  # tensors without a version are written as ever
        held, pages = x.clone(), pool.clone()
        assert torch.equal(rope(held, p, out=held), rope(x, p))
        certex.append_pages(x, x, pages, pages.clone(), table, p)
    certex.append_pages(x, x, pages, pages.clone(), table, p)
    assert pages.is_inference()


def test_out_that_requires_a_gradient_is_refused(gpu):
    """Neither a leaf nor a result of the graph is overwritten behind autograd's back."""
    rope = certex.Rotary(64)
    x, p = rand(5, 2, 64), torch.arange(5, device="cuda")
    leaf = rand(5, 2, 64, seed=1).requires_grad_()
    before = leaf.detach().clone()
    for out in (leaf, leaf * 2.0, leaf[:]):
        with pytest.raises(ValueError, match="out must not require a gradient"):
            rope(x, p, out=out)
    assert torch.equal(leaf, before)
    with torch.no_grad():  # as torch's own in-place operators go
        rope(x, p, out=leaf)
    assert torch.equal(leaf.detach(), rope(x, p)) and leaf._version == 1
