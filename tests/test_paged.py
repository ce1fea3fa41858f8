"""The attention operators without a GPU: frequencies against their formulas, refusals of the Python functions and of
the C entry points."""

import ctypes
import math
import os
import subprocess

import pytest
import torch

import libcertex_amd as certex
from libcertex_amd import _capi as C


def test_plain_frequencies():
    f = certex.Rotary(96, rotary_dim=40, base=500_000.0).frequencies
    want = [500_000.0 ** (-2 * i / 40) for i in range(20)]
    assert torch.allclose(f, torch.tensor(want, dtype=torch.float64), rtol=1e-14, atol=0)
    assert certex.Rotary(96).magnitude == 1.0 and certex.Rotary(96, magnitude=1.25).magnitude == 1.25


def test_scaled_frequencies():
    r, s, L = 64, 4.0, 2048
    f = certex.Rotary(r).frequencies
    linear = certex.Rotary(r, scaling="linear", factor=s)
    assert torch.allclose(linear.frequencies, f / s, rtol=1e-14, atol=0) and linear.magnitude == 1.0
    base = certex.Rotary(r, scaling="base", factor=s).frequencies
    stretched = 10000.0 * s ** (r / (r - 2))
    want = torch.tensor([stretched ** (-2 * i / r) for i in range(r // 2)], dtype=torch.float64)
    assert torch.allclose(base, want, rtol=1e-13, atol=0)
    assert base[0] == 1.0 and math.isclose(base[-1], f[-1] / s, rel_tol=1e-12)  # the slowest pair is interpolated by s
    ramp = certex.Rotary(r, scaling="ramp", factor=s, original_length=L, ramp=(1, 32))
    turns = L * f / (2 * math.pi)
    g = ((turns - 1) / 31).clamp(0, 1)
    assert torch.allclose(ramp.frequencies, f * (g + (1 - g) / s), rtol=1e-13, atol=0)
    assert torch.equal(ramp.frequencies[turns > 32], f[turns > 32]) and (g == 0).any() and (g == 1).any()
    assert math.isclose(ramp.magnitude, 0.1 * math.log(s) + 1, rel_tol=1e-15)
    assert certex.Rotary(r, scaling="ramp", factor=s, magnitude=1.0).magnitude == 1.0


@pytest.mark.parametrize("kw", [
    dict(head_dim=63), dict(head_dim=64, rotary_dim=7), dict(head_dim=64, rotary_dim=66), dict(head_dim=64, rotary_dim=0),
    dict(head_dim=64, layout="pairs"), dict(head_dim=64, scaling="log"), dict(head_dim=64, base=0.5),
    dict(head_dim=64, base=float("nan")), dict(head_dim=64, scaling="linear", factor=0.5),
    dict(head_dim=64, scaling="ramp", factor=2, ramp=(4, 4)), dict(head_dim=64, scaling="ramp", factor=2, original_length=0),
    dict(head_dim=2, scaling="base", factor=2), dict(head_dim=64, magnitude=0.0), dict(head_dim=64, magnitude=float("inf")),
])
def test_rotary_refusals(kw):
    with pytest.raises(ValueError):
        certex.Rotary(**kw)


def test_host_tensors_are_refused():
    x = torch.zeros(3, 2, 8)
    i = torch.zeros(3, dtype=torch.int32)
    pool, table = torch.zeros(2, 8, 2, 8), torch.zeros(3, 2, dtype=torch.int32)
    calls = [
        lambda: certex.Rotary(8)(x, i),
        lambda: certex.append_pages(x, x, pool, pool, table, i),
        lambda: certex.paged_attention(x, pool, pool, table, i),
        lambda: certex.selected_attention(x, x.long(), torch.zeros(2, 5, 8), 1.0),
    ]
    for call in calls:
        with pytest.raises(ValueError, match="GPU"):
            call()


def _tensor(shape, dtype, device=C.kDLROCM, strides=None):
    """A DLManagedTensor of no memory that is ever read."""
    m = C.DLManagedTensor()
    m.shape_ = (ctypes.c_int64 * len(shape))(*shape)
    m.strides_ = None if strides is None else (ctypes.c_int64 * len(shape))(*strides)
    code, bits = C._DL[dtype]
    m.dl_tensor = C.DLTensor(ctypes.c_void_p(4096), C.DLDevice(device, 0), len(shape), C.DLDataType(code, bits, 1),
                             ctypes.cast(m.shape_, ctypes.POINTER(ctypes.c_int64)),
                             None if strides is None else ctypes.cast(m.strides_, ctypes.POINTER(ctypes.c_int64)), 0)
    return m


def _need(q=(2, 8, 64), k=(4, 16, 2, 64), v=(4, 16, 2, 64), table=(2, 2), dtype=torch.float16, k_type=None, window=0,
          table_type=torch.int32, device=C.kDLROCM, strides=None):
    t = [_tensor(q, dtype, device), _tensor(k, k_type or dtype, strides=strides), _tensor(v, dtype),
         _tensor(table, table_type)]
    out = ctypes.c_int64()
    C.check(C.lib().cuvsCertexPagedAttentionWorkspace(*[ctypes.addressof(x) for x in t], window, ctypes.byref(out)))
    return out.value


def test_attention_checks():
    """The checks that the attention call and its workspace query share need no device."""
    assert _need() >= 0 and _need(q=(2, 6, 33), k=(4, 8, 3, 33), v=(4, 8, 3, 256)) >= 0
    for kw, match in [
        (dict(q=(2, 8, 63)), "same head dimension"), (dict(q=(2, 7, 64)), "multiple of the key heads"),
        (dict(q=(3, 8, 64)), "one row per sequence"), (dict(k=(4, 12, 2, 64), v=(4, 12, 2, 64)), "multiple of 8"),
        (dict(v=(4, 8, 2, 64)), "v_pages must have shape"), (dict(v=(4, 16, 2, 257)), "between 1 and 256"),
        (dict(q=(2, 8, 272), k=(4, 16, 2, 272)), "between 1 and 256"), (dict(k_type=torch.bfloat16), "element type"),
        (dict(dtype=torch.int32), "float32, float16 or bfloat16"), (dict(table_type=torch.int64), "must be int32"),
        (dict(device=C.kDLCPU), "device memory"), (dict(window=-1), "window"), (dict(q=(2, 8, 64, 1)), "3 dimensions"),
        (dict(k=(4, 16, 0, 64), v=(4, 16, 0, 64)), "multiple of the key heads"),
        (dict(strides=(2048, 128, 64, 2)), "dense in its last dimension"), (dict(table=(2, 2, 1)), "2 dimensions"),
        (dict(table=(2, 1 << 28)), "fewer than 2\\^31"),
    ]:
        with pytest.raises(ValueError, match=match):
            _need(**kw)


def test_misaligned_data_is_refused():
    t = [_tensor((2, 8, 64), torch.float16), *[_tensor((4, 16, 2, 64), torch.float16) for _ in range(2)],
         _tensor((2, 2), torch.int32)]
    out = ctypes.c_int64()
    for bad in range(4):
        for x in t:
            x.dl_tensor.byte_offset = 0
        t[bad].dl_tensor.byte_offset = 1
        with pytest.raises(ValueError, match="multiple of its element size"):
            C.check(C.lib().cuvsCertexPagedAttentionWorkspace(*[ctypes.addressof(x) for x in t], 0, ctypes.byref(out)))


def test_null_arguments_are_errors():
    L = C.lib()
    n = ctypes.c_int64()
    with pytest.raises(ValueError, match="q is NULL"):
        C.check(L.cuvsCertexPagedAttentionWorkspace(None, None, None, None, 0, ctypes.byref(n)))
    with pytest.raises(ValueError, match="NULL"):
        C.check(L.cuvsCertexSelectedAttentionWorkspace(None, None, None, None))
    with pytest.raises(ValueError, match="resources handle is NULL"):
        C.check(L.cuvsCertexRotate(0, 0, None, None, None, False))
    with pytest.raises(ValueError, match="resources handle is NULL"):
        C.check(L.cuvsCertexAppendPages(0, 0, *[None] * 9))
    with pytest.raises(ValueError, match="resources handle is NULL"):
        C.check(L.cuvsCertexSelectedAttention(0, *[None] * 4, 1.0, *[None] * 3))
    assert L.cuvsCertexRotaryDestroy(0) == C.CUVS_SUCCESS


def test_selection_checks():
    def need(scores=(4, 3, 5), values=(2, 9, 64), table=None, dtype=torch.float32):
        t = [_tensor(scores, dtype), _tensor(values, torch.bfloat16)]
        at = [ctypes.addressof(x) for x in t]
        keep = _tensor(table, torch.int32) if table else None
        out = ctypes.c_int64()
        C.check(C.lib().cuvsCertexSelectedAttentionWorkspace(*at, ctypes.addressof(keep) if keep else None,
                                                             ctypes.byref(out)))
        return out.value

    assert need() >= 0 and need(values=(6, 16, 2, 64), table=(3,)) >= 0
    for kw, match in [
        (dict(scores=(5, 3, 5)), "multiple of the value heads"), (dict(values=(2, 9, 300)), "between 1 and 256"),
        (dict(values=(6, 16, 2, 64)), "3 dimensions"), (dict(table=(3,)), "4 dimensions"),
        (dict(dtype=torch.float16), "scores must be float32"), (dict(scores=(4, 5)), "3 dimensions"),
    ]:
        with pytest.raises(ValueError, match=match):
            need(**kw)


def test_header_is_c():
    """certex_attention.h compiles as C99, warnings as errors."""
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    source = "#include <cuvs/neighbors/certex_attention.h>\nint main(void) { return CERTEX_ROTARY_HALF; }\n"
    r = subprocess.run(["gcc", "-std=c99", "-Wall", "-Wextra", "-Werror", "-fsyntax-only", "-I", include, "-x", "c", "-"],
                       input=source, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
