"""Attention operators next to the key cache, over the C API (include/cuvs/neighbors/certex_attention.h).

Rotary turns queries and keys by their positions; append_pages writes keys (turned on the way) and values
into a paged cache; paged_attention is the attention of one new token of every sequence over its pages;
selected_attention is the attention over the top k that KeyCache.topk returned. The reference has
no counterpart: its attention support ends at the ids and scores (certex/attention.py:84-106).

A paged cache is two pools, keys (n_pages, page_size, n_kv_heads, head_dim) and values (the same with their own
dimension), and a page table (n_sequences, n) of int32: position p of sequence s is slot p % page_size of
page table[s, p // page_size]. The program that schedules the sequences owns the pools, the table and the lengths;
the pools may be views of any strides with a dense last dimension. The calls run on torch's current
stream, read nothing back to the host and allocate from torch, so a graph capture records them.
"""

import ctypes
import threading

import torch

from . import _capi as C
from .index import _require

_ROWS = frozenset((torch.float32, torch.float16, torch.bfloat16))
_INTS = (torch.int32, torch.int64)
_LAYOUTS = {"half": 0, "interleaved": 1}
_SCALINGS = {None: 0, "linear": 1, "base": 2, "ramp": 3}


def _refuse_rows(t, what, ndim, like):
    """Why t is no row tensor of these dimensions (nothing for a subclass that is one)."""
    _require(isinstance(t, torch.Tensor) and t.is_cuda, f"{what} must be a GPU tensor")
    if like is None:
        _require(t.dtype in _ROWS, f"{what} must be float32, float16 or bfloat16, not {t.dtype}")
    else:
        _require(t.dtype == like.dtype, f"{what} must be {like.dtype} as the other tensors, not {t.dtype}")
    _require(t.ndim == ndim, f"{what} must have {ndim} dimensions, not shape {tuple(t.shape)}")


def _rows(t, what, ndim, like=None):
    """A row tensor on the GPU of one of the element types (of `like`'s, if given). The checks come once in one
    expression: a call that passes spends a fraction of a microsecond on them."""
    if not (type(t) is torch.Tensor and t.is_cuda and t.ndim == ndim
            and (t.dtype in _ROWS if like is None else t.dtype == like.dtype)):
        _refuse_rows(t, what, ndim, like)
    return t


def _read(t, what, ndim, like=None):
    """A row tensor that is only read: one whose last dimension has gaps is copied."""
    t = _rows(t, what, ndim, like)
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _ints(t, what, dtypes=_INTS):
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype in dtypes):
        raise ValueError(f"{what} must be a GPU tensor of " + " or ".join(str(d) for d in dtypes))
    return t if t.is_contiguous() else t.contiguous()


def _no_gradient(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError("this operator has no gradient: call it under torch.no_grad()")


def _output(like, shape):
    """A dense tensor of like's type and device."""
    return torch.empty_like(like) if like.is_contiguous() and like.shape == shape else like.new_empty(shape)


class _Rotate(torch.autograd.Function):
    """The rotation is linear and its matrix times the magnitude orthogonal: the gradient is the
    transposed rotation of the output's gradient."""

    @staticmethod
    def forward(ctx, x, positions, rope, transpose):
        ctx.save_for_backward(positions)
        ctx.rope, ctx.transpose = rope, transpose
        return rope._rotate(x, positions, transpose, None)

    @staticmethod
    def backward(ctx, dy):
        (positions,) = ctx.saved_tensors
        if torch.is_grad_enabled():  # a gradient of the gradient was asked for
            return _Rotate.apply(dy, positions, ctx.rope, not ctx.transpose), None, None, None
        return ctx.rope._rotate(dy, positions, not ctx.transpose, None), None, None, None


class Rotary:
    """The rotation of queries and keys by their positions.

        rope = certex.Rotary(128)
        q = rope(q, positions)           # q (tokens, heads, 128), positions (tokens,)

    The pair (a, b) of position p and frequency f becomes magnitude * (a cos pf - b sin pf, a sin pf + b cos pf),
    f_i = base^(-2 i / rotary_dim). Pairs are (i, i + rotary_dim / 2) in the "half" layout and (2 i, 2 i + 1) in the
    "interleaved" one; elements of a head past rotary_dim (default: all of head_dim) are copied. Long contexts
    scale the frequencies: "linear" divides them by `factor`; "base" takes the base times
    factor^(rotary_dim / (rotary_dim - 2)); "ramp" keeps pairs that turn more than ramp[1] times within original_length
    positions, divides those that turn less than ramp[0] times, and blends between, with the magnitude
    0.1 ln(factor) + 1 unless given. Any position goes: its product with the frequency (a double) is reduced to a turn
    exactly, in 64-bit fixed point. The first use on a GPU puts the frequencies there, which waits for the GPU: before a
    graph is recorded, call the rotation once.
    """

    def __init__(self, head_dim, rotary_dim=None, base=10000.0, layout="half", scaling=None, factor=1.0,
                 original_length=8192, ramp=(1.0, 32.0), magnitude=None):
        _require(layout in _LAYOUTS, f"layout must be one of {tuple(_LAYOUTS)}, not {layout!r}")
        _require(scaling in _SCALINGS, f"scaling must be one of {tuple(_SCALINGS)}, not {scaling!r}")
        self.head_dim = int(head_dim)
        self.rotary_dim = self.head_dim if rotary_dim is None else int(rotary_dim)
        _require(2 <= self.rotary_dim <= self.head_dim and self.rotary_dim % 2 == 0,
                 f"rotary_dim must be even and between 2 and {self.head_dim}, not {self.rotary_dim}")
        _require(magnitude is None or magnitude > 0, "the magnitude must be positive")
        self._handles, self._lock = {}, threading.Lock()
        p = ctypes.POINTER(C.RotaryParams)()
        C.check(C.lib().cuvsCertexRotaryParamsCreate(ctypes.byref(p)))
        c = p.contents
        self._params = C.RotaryParams(self.rotary_dim, _LAYOUTS[layout], float(base), _SCALINGS[scaling], float(factor),
                                      float(original_length), float(ramp[0]), float(ramp[1]),
                                      c.magnitude if magnitude is None else float(magnitude))
        C.check(C.lib().cuvsCertexRotaryParamsDestroy(p))
        f, m = (ctypes.c_double * (self.rotary_dim // 2))(), ctypes.c_double()
        C.check(C.lib().cuvsCertexRotaryFrequencies(ctypes.byref(self._params), f, ctypes.byref(m)))
        self.frequencies, self.magnitude = torch.tensor(list(f), dtype=torch.float64), m.value  # radians per position

    def _handle(self, device):
        """The frequencies on a GPU (kept from the first use there on)."""
        h = self._handles.get(device)
        if h is None:
            with self._lock:
                h = self._handles.get(device)
                if h is None:
                    out = ctypes.c_size_t()
                    C.check(C.lib().cuvsCertexRotaryCreate(C.stream_resources(), ctypes.byref(self._params), ctypes.byref(out)))
                    h = self._handles[device] = out.value
        return h

    def __del__(self):
        try:
            for h in self._handles.values():
                C.lib().cuvsCertexRotaryDestroy(h)
        except Exception:  # interpreter shutdown
            pass

    def __call__(self, x, positions, transpose=False, out=None):
        """x (tokens, heads, head_dim) or (batch, tokens, heads, head_dim), rotated by positions (tokens,) or (batch,
        tokens): a tensor of its own, or `out` (which may be x). transpose: by the negative angle. Differentiable
        in x (without out)."""
        if x.requires_grad and torch.is_grad_enabled():
            _require(out is None, "a rotation that is differentiated takes no out")
            return _Rotate.apply(x, positions, self, bool(transpose))
        return self._rotate(x, positions, bool(transpose), out)

    def _rotate(self, x, positions, transpose, out):
        if not (isinstance(x, torch.Tensor) and x.ndim in (3, 4) and x.shape[-1] == self.head_dim):
            raise ValueError(f"x must be a tensor (tokens, heads, {self.head_dim}) or (batch, tokens, heads, {self.head_dim})")
        x = _read(x, "x", x.ndim)
        positions = _ints(positions, "positions")
        if positions.shape != x.shape[:-2]:
            raise ValueError(f"positions must have shape {tuple(x.shape[:-2])}, one entry per token")
        y = torch.empty_like(x) if out is None else _rows(out, "out", x.ndim, x)
        if out is None and y.stride(-1) != 1:  # a dense tensor in another order of dimensions
            y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        _require(y.shape == x.shape, "out must have the shape of x")
        C.check(C.lib().cuvsCertexRotate(C.stream_resources(), self._handle(x.get_device()), *C.describe(0, x, positions, y),
                                         transpose))
        return y


def append_pages(k, v, k_pages, v_pages, page_table, positions, sequences=None, rotary=None, q=None):
    """Write token t's keys k[t] (n_kv_heads, head_dim) and values v[t] to position positions[t] of sequence
    sequences[t] (default: t) of the paged cache, in place; `rotary` turns the keys on the way. With q (tokens, n_heads,
    head_dim) the same launch rotates the queries, which are returned (else None).

    A token with a negative position or sequence is padding and is not written; neither is one whose page the
    table does not hold (an entry outside the pool, such as -1). Positions of one call are to be distinct."""
    k = _read(k, "k", 3)
    v = _read(v, "v", 3, k)
    _rows(k_pages, "k_pages", 4, k)
    _rows(v_pages, "v_pages", 4, k)
    _no_gradient(k, v, q, k_pages, v_pages)
    table = _ints(page_table, "page_table", (torch.int32,))
    positions = _ints(positions, "positions")
    out = None
    if sequences is not None:
        sequences = _ints(sequences, "sequences")
    if q is not None:
        q = _read(q, "q", 3, k)
        out = _output(q, q.shape)
    if rotary is not None and rotary.head_dim != k.shape[-1]:
        raise ValueError(f"this rotation is of heads of {rotary.head_dim}, not {k.shape[-1]}")
    C.check(C.lib().cuvsCertexAppendPages(
        C.stream_resources(), 0 if rotary is None else rotary._handle(k.get_device()),
        *C.describe(0, k, v, k_pages, v_pages, table, positions, sequences, q, out)))
    return out


def paged_attention(q, k_pages, v_pages, page_table, lengths, scale=None, window=None, return_lse=False):
    """Attention of one new token of every sequence over its pages: q (n_sequences, n_heads, head_dim) gives
    (n_sequences, n_heads, value_dim), softmax(scale q k) v over the positions below lengths[s] (the last `window` of
    them, if given); query head h reads key head h // (n_heads / n_kv_heads). scale defaults to head_dim ** -0.5.

    A sequence of length 0 gives zeros. Lengths past the table's pages are cut to them, positions whose page the
    table does not hold do not count, and slots past a length are never used, whatever they hold. With
    return_lse also the logarithm of the softmax's denominator (float32, -inf for an empty row), which
    joins the outputs of two calls over different positions. A cache holds head dimensions up to 256 and
    pages of a multiple of 8 positions."""
    q = _read(q, "q", 3)
    _rows(k_pages, "k_pages", 4, q)
    _rows(v_pages, "v_pages", 4, q)
    _no_gradient(q, k_pages, v_pages)
    table = _ints(page_table, "page_table", (torch.int32,))
    lengths = _ints(lengths, "lengths")
    if window is not None and window < 1:
        raise ValueError(f"the window must be at least 1, not {window}")
    window = 0 if window is None else int(window)
    out = _output(q, (*q.shape[:2], v_pages.shape[3]))
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device) if return_lse else None
    L, need = C.lib(), ctypes.c_int64()
    qv, kv, vv, tv, lv, ov, ev = C.describe(0, q, k_pages, v_pages, table, lengths, out, lse)
    C.check(L.cuvsCertexPagedAttentionWorkspace(qv, kv, vv, tv, window, ctypes.byref(need)))
    work = q.new_empty(need.value, dtype=torch.uint8) if need.value else None
    C.check(L.cuvsCertexPagedAttention(C.stream_resources(), qv, kv, vv, tv, lv,
                                       q.shape[2] ** -0.5 if scale is None else float(scale), window,
                                       *C.describe(7, work), ov, ev))
    return (out, lse) if return_lse else out


def selected_attention(scores, ids, values, scale, page_table=None, return_lse=False):
    """Attention over a selected top k, as KeyCache.topk returns it: scores (float32) and ids (n_heads, queries, k) or
    (n_heads, k) give (n_heads, queries, value_dim) or (n_heads, value_dim), softmax(scale * scores) times the values of the
    ids. values is (n_kv_heads, n, value_dim), or with page_table (one sequence's pages, int32 (n,)) a pool of pages (n_pages,
    page_size, n_kv_heads, value_dim). Query head h reads value head h // (n_heads / n_kv_heads).

    Ids outside the values (-1 marks a missing neighbour) and scores of -inf do not count; a row of none gives zeros.
    With return_lse also the logarithm of the softmax's denominator (float32, -inf for an empty row)."""
    _require(isinstance(scores, torch.Tensor) and scores.is_cuda and scores.dtype == torch.float32,
             "scores must be a float32 GPU tensor")
    ids = _ints(ids, "ids")
    if scores.ndim not in (2, 3) or scores.shape != ids.shape:
        raise ValueError(f"scores and ids must have one shape (n_heads, queries, k) or (n_heads, k), not "
                         f"{tuple(scores.shape)} and {tuple(ids.shape)}")
    values = _read(values, "values", 3 if page_table is None else 4)
    _no_gradient(scores, values)
    if page_table is not None:
        page_table = _ints(page_table, "page_table", (torch.int32,))
        _require(page_table.ndim == 1, "page_table must be one sequence's pages, of shape (n,)")
    single = scores.ndim == 2
    if single:
        scores, ids = scores[:, None], ids[:, None]
    scores = scores.contiguous()
    out = values.new_empty((*scores.shape[:2], values.shape[-1]))
    lse = torch.empty(scores.shape[:2], dtype=torch.float32, device=values.device) if return_lse else None
    L, need = C.lib(), ctypes.c_int64()
    sv, iv, vv, tv, ov, ev = C.describe(0, scores, ids, values, page_table, out, lse)
    C.check(L.cuvsCertexSelectedAttentionWorkspace(sv, vv, tv, ctypes.byref(need)))
    work = values.new_empty(need.value, dtype=torch.uint8) if need.value else None
    C.check(L.cuvsCertexSelectedAttention(C.stream_resources(), sv, iv, vv, tv, float(scale), *C.describe(6, work), ov, ev))
    if single:
        out, lse = out[:, 0], None if lse is None else lse[:, 0]
    return (out, lse) if return_lse else out
