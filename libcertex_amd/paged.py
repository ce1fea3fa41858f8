"""Attention operators next to the key cache, over the C API (include/cuvs/neighbors/certex_attention.h).

Rotary turns queries and keys by their positions; append_pages writes keys (turned on the way) and values
into a paged cache; paged_attention is the attention of one new token of every sequence over its pages, prompt_attention that of many;
selected_attention is the attention over the top k that KeyCache.topk returned. PackedPages is a paged cache of 4-bit elements. The reference has
no counterpart: its attention support ends at the ids and scores (certex/attention.py:84-106).

A paged cache is two pools, keys (n_pages, page_size, n_kv_heads, head_dim) and values (the same with their own
dimension), and a page table (n_sequences, n) of int32: position p of sequence s is slot p % page_size of
page table[s, p // page_size]. The program that schedules the sequences owns the pools, the table and the lengths;
the pools may be views of any strides with a dense last dimension. The calls run on torch's current
stream, read nothing back to the host and allocate from torch, so a graph capture records them. As for an Index their tensors
are on the current GPU (torch.cuda.device chooses it); tensors of another one are an error. Only the rotation has a
gradient; tensors that ask for another, or carry a tangent of forward-mode differentiation, are refused. What a call
writes in place (out, k_pages, v_pages) changes its version, so that a backward pass that saved it before raises.
"""

import ctypes
import threading

import torch

from . import _capi as C
from .index import _require

_LAYOUTS = {"half": 0, "interleaved": 1}
_SCALINGS = {None: 0, "linear": 1, "base": 2, "ramp": 3}


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
    exactly, in 64-bit fixed point. The frequencies are put on the current GPU when the rotation is made (if
    the program has used a GPU by then) and on others at the first use there, which waits for that GPU: before a graph
    is recorded, not in it. A graph that rotates reads them there: keep the rotation as long as the graph.
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
        self._handles, self._lock = {}, threading.Lock()  # by GPU
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
        if torch.cuda.is_initialized() and not torch.cuda.is_current_stream_capturing():
            self._on(torch.cuda.current_device())

    def _on(self, device):
        """The frequencies on a GPU, as the extension's capsule (made at the first use, or with the rotation)."""
        h = self._handles.get(device)
        if h is None:
            with self._lock:
                h = self._handles.get(device)
                if h is None:
                    out = ctypes.c_size_t()
                    with torch.cuda.device(device):
                        C.check(C.lib().cuvsCertexRotaryCreate(C.stream_resources(), ctypes.byref(self._params),
                                                               ctypes.byref(out)))
                    h = self._handles[device] = C.operators().own(out.value)
        return h

    def _handle(self, like):
        _require(isinstance(like, torch.Tensor) and like.is_cuda, "rotated tensors must be GPU tensors")
        return self._on(like.get_device())

    def __call__(self, x, positions, transpose=False, out=None):
        """x (tokens, heads, head_dim) or (batch, tokens, heads, head_dim), rotated by positions (tokens,) or (batch,
        tokens): a tensor of its own, or `out` (which may be x, and else shares no memory with it). transpose: by the negative angle. Differentiable
        in x (without out)."""
        return C.operators().rotate(self._handle(x), self.head_dim, x, positions, transpose, out)


def append_pages(k, v, k_pages, v_pages, page_table, positions, sequences=None, rotary=None, q=None):
    """Write token t's keys k[t] (n_kv_heads, head_dim) and values v[t] to position positions[t] of sequence
    sequences[t] (default: t) of the paged cache, in place; `rotary` turns the keys on the way. With q (tokens, n_heads,
    head_dim) the same launch rotates the queries, which are returned (else None).

    A token with a negative position or sequence is padding and is not written; neither is one whose page the
    table does not hold (an entry outside the pool, such as -1). The tokens of one call are to have positions of their own: a slot that
    several name ends with elements of any of them mixed."""
    return C.operators().append(None if rotary is None else rotary._handle(k), 0 if rotary is None else rotary.head_dim, k, v,
                                k_pages, v_pages, page_table, positions, sequences, q)


def paged_attention(q, k_pages, v_pages, page_table, lengths, scale=None, window=None, return_lse=False, cap=None,
                    slopes=None):
    """Attention of one new token of every sequence over its pages: q (n_sequences, n_heads, head_dim) gives
    (n_sequences, n_heads, value_dim), softmax(scale q k) v over the positions below lengths[s] (the last `window` of
    them, if given); query head h reads key head h // (n_heads / n_kv_heads). scale defaults to head_dim ** -0.5.

    With a cap the scores are cap * tanh(scale q k / cap); with slopes (float32 (n_heads,), finite) a score loses slopes[h] times the
    distance of its key from the new token, after the cap.

    A sequence of length 0 gives zeros. Lengths past the table's pages are cut to them, positions whose page the
    table does not hold do not count, and slots past a length are never used, whatever they hold; an
    infinite value that counts, however little it weighs, makes its column of the output infinite or NaN. With
    return_lse also the logarithm of the softmax's denominator (float32, -inf for an empty row), which
    joins the outputs of two calls over different positions. A cache holds head dimensions up to 256 and
    pages of a multiple of 8 positions."""
    return C.operators().attend(q, k_pages, v_pages, page_table, lengths, scale, window, return_lse, cap, slopes)


def prompt_attention(q, k_pages, v_pages, page_table, lengths, first, scale=None, window=None, prefix=None, cap=None,
                     slopes=None, return_lse=False):
    """Attention of the new tokens of every sequence over its pages, where append_pages has put their keys and values: q
    (tokens, n_heads, head_dim) gives (tokens, n_heads, value_dim). Sequence s has the tokens q[first[s] : first[s + 1]] (first:
    (n_sequences + 1,), not decreasing), which are the last of its lengths[s] positions: a whole prompt, a piece of one
    behind what the cache holds, or one new token.

    A token at position p sees the positions t <= p of its sequence, and with prefix (n_sequences,) those below
    prefix[s] too; with a window only those less than `window` before it (t > p - window). Scores, cap and slopes as in
    paged_attention, slopes times |p - t|.

    Tokens that see nothing (more tokens than the length has positions) and tokens of no sequence give zeros. Lengths, missing
    pages, unused slots, return_lse and the cache's sizes as in paged_attention; an infinite value shows in the rows that see it."""
    return C.operators().prompt(q, k_pages, v_pages, page_table, lengths, first, scale, window, prefix, cap, slopes,
                                return_lse)


class PackedPages:
    """A paged cache of 4-bit keys and values, in 9/32 of what 16-bit pages take (heads of 64, 128, 192 and 256 elements;
    others are padded to 64, 96, 128, 192 or 256).

        pages = certex.PackedPages(n_pages, page_size=64, n_kv_heads=8, head_dim=128)
        pages.append(k, v, table, positions, sequences, rotary=rope)
        out = pages.attend(q, table, lengths)

    Of every 64 consecutive elements x of a key or value (the last ones of a head fewer): an offset o, the float16 nearest to their
    minimum, a scale s, the float16 nearest to the float32 product (maximum - o) * float32(1 / 15), and codes round((x - o) / s) in
    0..15 (half to even; all 0 where s is 0), which stand for o + s code. o and s are cut to float16's finite range; NaN makes its 64 elements
    NaN. Page tables, positions and lengths are those of append_pages and paged_attention, pages of a multiple of 8 positions.

    `data` holds the pages, uint8 (n_pages, n_kv_heads, page_size / 8, record): pages can be copied in it, as
    data[new] = data[old], and a program may bring its own memory of that shape (contiguous, aligned to 16 bytes)."""

    def __init__(self, n_pages, page_size, n_kv_heads, head_dim, value_dim=None, data=None):
        self.page_size, self.n_kv_heads, self.head_dim = int(page_size), int(n_kv_heads), int(head_dim)
        self.value_dim = self.head_dim if value_dim is None else int(value_dim)
        _require(int(n_pages) >= 0 and self.n_kv_heads >= 1, "n_pages must not be negative and n_kv_heads positive")
        _require(self.page_size >= 8 and self.page_size % 8 == 0,
                 f"the page size must be a multiple of 8, not {self.page_size}")
        record = ctypes.c_int64()
        C.check(C.lib().cuvsCertexPackedRecord(self.head_dim, self.value_dim, ctypes.byref(record)))
        shape = (int(n_pages), self.n_kv_heads, self.page_size // 8, record.value)
        if data is None:
            data = torch.zeros(shape, dtype=torch.uint8, device="cuda")
        _require(isinstance(data, torch.Tensor) and data.is_cuda and data.dtype == torch.uint8 and data.is_contiguous()
                 and tuple(data.shape) == shape, f"data must be a contiguous uint8 GPU tensor of shape {shape}")
        self.data = data

    def append(self, k, v, page_table, positions, sequences=None, rotary=None):
        """As append_pages: token t's keys k[t] (n_kv_heads, head_dim), turned by `rotary` and rounded to their type, and values
        v[t] to position positions[t] of sequence sequences[t] (default: t), in 4 bits."""
        C.operators().pack(None if rotary is None else self._turn(rotary, k), self.head_dim, self.value_dim, k, v, self.data,
                           page_table, positions, sequences)

    def _turn(self, rotary, k):
        _require(rotary.head_dim == self.head_dim,
                 f"this rotation is of heads of {rotary.head_dim}, not {self.head_dim}")
        return rotary._handle(k)

    def read(self, page_table, positions, sequences=None, dtype=torch.bfloat16):
        """The keys (tokens, n_kv_heads, head_dim) and values that the pages hold at positions[t] of sequence sequences[t] (default:
        t), rounded to dtype; zeros where the table does not hold the page."""
        _require(isinstance(dtype, torch.dtype), f"dtype must be a torch.dtype, not {dtype!r}")
        return C.operators().unpack(self.head_dim, self.value_dim, self.data, page_table, positions, sequences,
                                    torch.empty(0, dtype=dtype))

    def attend(self, q, page_table, lengths, scale=None, window=None, return_lse=False, cap=None, slopes=None):
        """As paged_attention: q (n_sequences, n_heads, head_dim) of any element type gives (n_sequences, n_heads, value_dim)
        of the same. Groups of 64 values that are more than 2^14 times smaller than others of their head lose precision: at 2^26
        float16's is left."""
        return C.operators().attend_packed(self.head_dim, self.value_dim, q, self.data, page_table, lengths, scale, window, cap,
                                           slopes, return_lse)


def selected_attention(scores, ids, values, scale, page_table=None, return_lse=False):
    """Attention over a selected top k, as KeyCache.topk returns it: scores (float32) and ids (n_heads, queries, k) or
    (n_heads, k) give (n_heads, queries, value_dim) or (n_heads, value_dim), softmax(scale * scores) times the values of the
    ids. values is (n_kv_heads, n, value_dim), or with page_table (one sequence's pages, int32 (n,)) a pool of pages (n_pages,
    page_size, n_kv_heads, value_dim). Query head h reads value head h // (n_heads / n_kv_heads).

    Ids outside the values (-1 marks a missing neighbour) and scores of -inf do not count; a row of none gives zeros.
    An infinite value that counts, however little it weighs, makes its column of the output infinite or NaN.
    With return_lse also the logarithm of the softmax's denominator (float32, -inf for an empty row)."""
    return C.operators().select(scores, ids, values, scale, page_table, return_lse)
